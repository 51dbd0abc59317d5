"""MxDecodeStep: each call of a step against the 64-bit form of what that call was given, over steps of a serving loop, and a
captured step against the launched one, bit for bit. The bars are the operators' own."""
import functools

import pytest
import torch

import intent_amd as intent
from intent_amd.examples.kernels.streaming import mx_cache
from intent_amd.examples.programs.mx_decode_step import MxDecodeStep
from tests import plain64
from tests import test_gpu_linear_mxfp4 as linear
from tests import test_gpu_mx_decode as decode
from tests import test_gpu_norm_rope as norm
from tests.gpu_util import announce
from tests.test_gpu_mx_cache import cache, i32, tables

pytestmark = pytest.mark.gpu

EPS = 1e-6


def layer(seed, dtype, lengths, steps, page, q_heads, kv_heads, d, pairs, hidden, head_major, device):
    """The arguments of a step, whose cache holds `lengths` rows per sequence (None: a sequence without pages)."""
    g = torch.Generator().manual_seed(seed)
    pages, offsets, indices = tables([0 if n is None else n + steps for n in lengths], page, g)
    x = torch.zeros((len(lengths), hidden), dtype=norm.TYPES[dtype], device=device)
    weights = [t.to(device) for n, k in (((q_heads + 2 * kv_heads) * d, hidden), (hidden, q_heads * d))
               for t in linear.case(seed + n, dtype, 1, n, k, 117, 121)[1:]]
    scales = (1 + 0.3 * torch.randn((2, d), generator=g)).to(device)
    cos, sin = (t.to(device) for t in norm.tables(pairs))
    held = (*cache(pages, page, kv_heads, d, head_major, device), *cache(pages, page, kv_heads, d, head_major, device))
    now = i32([0 if n is None else n for n in lengths], device)
    return dict(x=x, qkv_weight=weights[0], qkv_exponents=weights[1], out_weight=weights[2], out_exponents=weights[3],
                q_weight=scales[0], k_weight=scales[1], positions=now - 1, cos=cos, sin=sin, key_cache=held[0],
                key_exponents=held[1], value_cache=held[2], value_exponents=held[3],
                cu_seqlens=i32(range(len(lengths) + 1), device), page_offsets=i32(offsets, device),
                page_indices=indices.to(device), sequence_lengths=now, eps=EPS, scale=d ** -0.5)


def values(elements, exponents):
    return plain64.dequantise(elements.contiguous().float().cpu(), exponents.contiguous().cpu())


def prefill(case, dtype, g):
    """Rows of the lengths given go into the cache before the first step."""
    lengths = case["sequence_lengths"]
    cu = torch.zeros(len(lengths) + 1, dtype=torch.int32)
    cu[1:] = lengths.cpu().cumsum(0)
    shape = (int(cu[-1]), case["key_cache"].shape[2], case["key_cache"].shape[3])
    k, v = (torch.randn(shape, generator=g).to(norm.TYPES[dtype]).to(lengths.device) for _ in range(2))
    names = ("key_cache", "key_exponents", "value_cache", "value_exponents")
    intent.jit(getattr(mx_cache, f"paged_cache_append_{dtype}"), backend="hip").run(
        k, v, *(case[n] for n in names), cu.to(lengths.device), case["page_offsets"], case["page_indices"], lengths)


CASES = [("bf16", [5, 16, 0, None], 16, 8, 2, 128, 64, 256, True, False), ("f16", [40, 1], 7, 6, 3, 64, 16, 192, False, True),
         ("bf16", [300, 2047, 63], 64, 16, 2, 128, 64, 512, True, False)]


@pytest.mark.parametrize("dtype,lengths,page,q_heads,kv_heads,d,pairs,hidden,head_major,interleaved", CASES)
def test_steps(device, dtype, lengths, page, q_heads, kv_heads, d, pairs, hidden, head_major, interleaved):
    announce("decode step", dtype, lengths, q_heads, kv_heads, d)
    steps, g = 3, torch.Generator().manual_seed(d + page)
    one = layer(1, dtype, lengths, steps, page, q_heads, kv_heads, d, pairs, hidden, head_major, device)
    prefill(one, dtype, g)
    two = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in one.items()}
    program = MxDecodeStep.from_jit(functools.partial(intent.jit, backend="hip"), dtype=dtype, head_group=q_heads // kv_heads,
                                    interleaved=interleaved)
    launched, captured = program.prepare(**one), program.prepare(**two)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        captured.launch()
    live = torch.tensor([n is not None for n in lengths])
    for step in range(steps):
        x = torch.randn(one["x"].shape, generator=g).to(norm.TYPES[dtype])
        for case in (one, two):
            case["x"].copy_(x)
            case["sequence_lengths"] += live.to(device).int()
            case["positions"] += 1
        launched.launch()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(launched.result(), captured.result())
        for name in ("key_cache", "key_exponents", "value_cache", "value_exponents"):
            assert torch.equal(one[name].view(torch.uint8), two[name].view(torch.uint8))
        qkv, (q, k), _, heads, out = (c.result() for c in launched.calls)
        linear.check(qkv, x, one["qkv_weight"].cpu(), one["qkv_exponents"].cpu(), dtype)
        rows = qkv.unflatten(1, (-1, d)).cpu()
        for got, first, weight in ((q, 0, one["q_weight"]), (k, q_heads, one["k_weight"])):
            given = rows[:, first:first + got.shape[1]]
            want, size = plain64.norm_rope(given, weight.cpu(), one["positions"].cpu(), one["cos"].cpu(), one["sin"].cpu(), EPS,
                                           interleaved)
            norm.close(got, want, size, dtype, 2.0 ** -18)
        keys, held = values(one["key_cache"], one["key_exponents"]), values(one["value_cache"], one["value_exponents"])
        offsets, indices, now = (one[n].cpu() for n in ("page_offsets", "page_indices", "sequence_lengths"))
        for s in live.nonzero().flatten().tolist():
            p = int(now[s]) - 1
            place = int(indices[offsets[s] + p // page]), p % page
            for cached, new in ((keys, k[s]), (held, rows[s, q_heads + kv_heads:])):
                assert torch.equal(cached[place], plain64.dequantise(*plain64.quantise(new.cpu())))
        decode.check(heads, q.cpu(), keys, held, offsets.tolist(), indices, now.tolist(), one["scale"], dtype)
        linear.check(out, heads.flatten(1).cpu(), one["out_weight"].cpu(), one["out_exponents"].cpu(), dtype)
        assert (heads[~live.to(device)] == 0).all() and (out[~live.to(device)] == 0).all()
    assert launched.kernel_count == 5
    names = [o.kernel.split("<")[0] for o in launched.observations]
    assert names == ["linear_few", "norm_rope_rows", "cache_append", "mx_decode", "linear_few"]
