"""Calls whose tensors have a layout that was bound before: other tensors, alignments, scalars, overlaps, devices and streams.
Each is compared bit for bit with the same call of a new kernel, or refused as that one refuses it."""
import gc
import weakref

import pytest
import torch

import intent_amd as intent
from tests import test_gpu_linear_mxfp4 as linear
from tests import test_gpu_norm_rope as norm
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu


def arguments(seed, device, tokens=9, q_heads=4, kv_heads=2, d=64, pairs=32):
    rows, weights, positions, cos, sin, *grads = norm.case(seed, "bf16", tokens, q_heads, kv_heads, d, pairs)
    rows = rows.to(device)
    return ([rows[:, :q_heads], rows[:, q_heads:q_heads + kv_heads], *weights.to(device), positions.to(device), cos.to(device),
             sin.to(device)], [t.to(device) for t in grads])


def test_other_tensors_and_scalars(device):
    announce("repeated layouts, other tensors")
    kept, back = norm.kernel("qk_norm_rope_bf16"), norm.kernel("qk_norm_rope_backward_bf16")
    for seed, eps in ((0, 1e-6), (1, 1e-6), (2, 0.25), (3, 0.25)):
        inputs, grads = arguments(seed, device)
        for got, want in ((kept.run(*inputs, eps), norm.kernel("qk_norm_rope_bf16").run(*inputs, eps)),
                          (back.run(*inputs, *grads, eps), norm.kernel("qk_norm_rope_backward_bf16").run(*inputs, *grads, eps))):
            for a, b in zip(got, want):
                assert torch.equal(a, b)
                assert a.data_ptr() not in [t.data_ptr() for t in (*inputs, *grads)]
    layouts = list(kept.artifacts[0].runtime._layouts)
    assert len(layouts) == 1


def test_alignment_and_strides_are_another_layout(device):
    announce("repeated layouts, alignment")
    kept = norm.kernel("qk_norm_rope_bf16")
    inputs, _ = arguments(4, device)
    want = kept.run(*inputs, norm.EPS)
    for shift in (1, 8):
        storage = torch.zeros(inputs[0].numel() + 16, dtype=torch.bfloat16, device=device)
        moved = storage[shift:shift + inputs[0].numel()].view(inputs[0].shape)
        moved.copy_(inputs[0])
        got = kept.run(moved, *inputs[1:], norm.EPS)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    turned = inputs[0].permute(2, 1, 0).contiguous().permute(2, 1, 0)          # inner stride not 1: staged
    for _ in range(2):
        got = kept.run(turned, *inputs[1:], norm.EPS)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals_stay(device):
    """What a first call is refused for, a later one of a known layout is refused for as well."""
    announce("repeated layouts, refusals")
    kept = norm.kernel("qk_norm_rope_bf16")
    inputs, _ = arguments(5, device)
    outs = [torch.empty_like(t, memory_format=torch.contiguous_format) for t in inputs[:2]]
    for _ in range(2):
        kept(*inputs, *outs, norm.EPS)
    same = torch.empty(outs[0].shape, dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError, match="overlap"):
        kept(same, *inputs[1:], same[:], outs[1], norm.EPS)
    block = torch.empty((18, *outs[0].shape[1:]), dtype=torch.bfloat16, device=device)
    inputs_at = [block[:9], *inputs[1:]]
    kept(*inputs_at, block[9:], outs[1], norm.EPS)
    with pytest.raises(ValueError, match="overlap"):
        kept(*inputs_at, block[4:13], outs[1], norm.EPS)
    with pytest.raises(TypeError):
        kept.run(inputs[0].half(), *inputs[1:], norm.EPS)
    with pytest.raises(ValueError):
        kept.run(*inputs[:4], inputs[4][:-1], *inputs[5:], norm.EPS)
    with pytest.raises(ValueError):
        kept.run(inputs[0].cpu(), *inputs[1:], norm.EPS)
    with pytest.raises(TypeError):
        kept.run(*inputs)
    with pytest.raises(TypeError):
        kept.run(inputs[0].tolist(), *inputs[1:], norm.EPS)


def test_nothing_outlives_its_call(device):
    announce("repeated layouts, lifetime")
    kept = linear.kernel("f16")
    seen = []
    for seed in range(3):
        x, weight, exponents = (t.to(device) for t in linear.case(seed, "f16", 3, 40, 96))
        out = kept.run(x, weight, exponents)
        seen += [weakref.ref(t) for t in (x, weight, exponents, out)]
    x, weight, exponents = (t.to(device) for t in linear.case(9, "f16", 5, 40, 96))
    kept.run(x, weight, exponents)                                             # the last launch's tensors are kept, no others
    del out
    gc.collect()
    x2, weight2, exponents2 = x.clone(), weight.clone(), exponents.clone()
    kept.run(x2, weight2, exponents2)
    gc.collect()
    assert not [r for r in seen if r() is not None]


def test_streams_and_capture(device):
    """A call of a known layout with a workspace on another stream, and into a graph replayed beside eager calls."""
    announce("repeated layouts, streams")
    kept = linear.kernel("bf16")
    cases = [[t.to(device) for t in linear.case(seed, "bf16", 20, 500, 2080)] for seed in range(3)]
    want = [linear.kernel("bf16").run(*c) for c in cases]
    kept.run(*cases[0])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = kept.run(*cases[1])
    side.synchronize()
    assert torch.equal(got, want[1])
    held = [t.clone() for t in cases[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kept.run(*held)
    for at in (1, 2, 0):
        for t, new in zip(held, cases[at]):
            t.copy_(new)
        graph.replay()
        eager = kept.run(*cases[(at + 1) % 3])
        torch.cuda.synchronize()
        assert torch.equal(out, want[at]) and torch.equal(eager, want[(at + 1) % 3])


def test_many_layouts(device):
    announce("repeated layouts, many")
    kept = linear.kernel("f16")
    _, weight, exponents = (t.to(device) for t in linear.case(1, "f16", 1, 24, 64))
    x = torch.randn((600, 64), device=device).half()
    for m in (*range(1, 600), 1, 300):
        got = kept.run(x[:m], weight, exponents)
        assert got.shape == (m, 24)
    assert len(kept.artifacts[0].runtime._layouts) <= 256
    linear.check(got, x[:300].cpu(), weight.cpu(), exponents.cpu(), "f16")
