"""Int8LayerStep: each call of a step against the 64-bit form of what that call was given, over steps of a serving loop, and a captured
step against the launched one, bit for bit. The bars are the operators' own."""
import functools

import pytest
import torch

import intent_amd as intent
from intent_amd.examples.programs.int8_layer_step import Int8LayerStep
from tests import prefix_bar
from tests import test_gpu_linear_i8 as linear
from tests import test_gpu_prefix_decode as decode
from tests import test_gpu_residual_norm as norm
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu

NUMBERS = (1.0, 0.5, 1e-6)


def weight(seed, n, k, biased, device):
    _, whole, _, scales, bias = linear.case(seed, 1, n, k, biased)
    return whole.to(device), (scales / 8).to(device), bias.to(device)


def step_of(seed, dtype, prefix, lengths, heads, kv_heads, d, ps, hidden, wide, device):
    given = decode.case(seed, dtype, prefix, lengths, heads, kv_heads, d, ps)
    g = torch.Generator().manual_seed(seed)
    norms = [[(1 + 0.2 * torch.randn((n,), generator=g)).to(device) for n in (post, hidden)] for post in (hidden, 0)]
    residual = torch.randn((len(lengths), hidden), generator=g).to(norm.TYPES[dtype]).to(device)
    return ([t.to(device) for t in given[:8]] + [given[8]] +
            [residual, weight(seed + 1, hidden, heads * d, True, device), weight(seed + 2, 2 * wide, hidden, False, device),
             weight(seed + 3, hidden, wide, True, device), norms[0], norms[1], *NUMBERS])


def checked(prepared, arguments, dtype):
    """Every call of the step against what it was given."""
    cpu = lambda tensors: [t.cpu() for t in tensors]  # noqa: E731
    attend, heads, project, middle, halves, gated, back, last = prepared.calls
    prefix_bar.check(attend.result(), *prefix_bar.bar(*cpu(arguments[:8]), arguments[8], dtype))
    want, want_scales = linear.quantised(attend.result().flatten(1).cpu())
    assert torch.equal(heads.result()[0].cpu().double(), want) and torch.equal(heads.result()[1].cpu(), want_scales)

    def product(call, rows, of):
        whole, scales, bias = cpu(of)
        elements, row_scales = cpu(rows)
        linear.check(call.result(), elements, whole, row_scales, scales, bias, dtype)

    none = torch.zeros(0)
    product(project, heads.result(), arguments[10])
    h, h_size, y, y_size = norm.plain(project.result().cpu(), arguments[9].cpu(), none, *cpu(arguments[13]), numbers=NUMBERS)
    norm.close(middle.result()[0], h, h_size, dtype)
    norm.check_i8(*middle.result()[1:], y, y_size, len(h))
    product(halves, middle.result()[1:], arguments[11])
    linear.check_gated(*gated.result(), *cpu(halves.result().chunk(2, 1)))
    product(back, gated.result(), arguments[12])
    h, h_size, y, y_size = norm.plain(back.result().cpu(), middle.result()[0].cpu(), none, *cpu(arguments[14]), numbers=NUMBERS)
    norm.close(last.result()[0], h, h_size, dtype)
    norm.close(last.result()[1], y, y_size, dtype)


CASES = [("bf16", 100, [5, 16, 0, 300], 8, 2, 128, 16, 256, 512), ("f16", 33, [40], 6, 3, 64, 7, 208, 336),
         ("bf16", 1500, [30] * 20, 16, 2, 128, 64, 1024, 2064)]


@pytest.mark.parametrize("dtype,prefix,lengths,heads,kv_heads,d,ps,hidden,wide", CASES)
def test_steps(device, dtype, prefix, lengths, heads, kv_heads, d, ps, hidden, wide):
    announce("int8 layer step", dtype, prefix, len(lengths), hidden)
    arguments = step_of(len(lengths), dtype, prefix, lengths, heads, kv_heads, d, ps, hidden, wide, device)
    program = Int8LayerStep.from_jit(functools.partial(intent.jit, backend="hip"), dtype=dtype, head_group=heads // kv_heads)
    prepared = program.prepare(*arguments)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prepared.launch()
    for step in range(3):
        arguments[0].copy_(arguments[0].roll(1, 0).neg())
        arguments[9].mul_(0.5)
        if step:
            arguments[7].sub_(1).clamp_(min=0)
        prepared.launch()
        torch.cuda.synchronize()
        checked(prepared, arguments, dtype)
        want = [t.clone() for t in prepared.result()]
        for t in prepared.result():
            t.zero_()
        graph.replay()
        fresh = program.run(*arguments)
        torch.cuda.synchronize()
        for a, b, c in zip(prepared.result(), want, fresh):
            assert torch.equal(a, b) and torch.equal(c, b)
    outputs = tuple(torch.empty_like(t) for t in prepared.result())
    program.prepare(*arguments, outputs=outputs).launch()
    assert all(torch.equal(a, b) for a, b in zip(outputs, want))
