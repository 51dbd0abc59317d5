"""paged_gqa_decode_prefix against its 64-bit form; the bar is that of prefix_bar.py."""
import pytest
import torch

import intent_amd as intent
from intent_amd.examples.kernels.streaming import prefix_decode
from tests import prefix_bar
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def kernel(dtype, group, **options):
    return intent.jit(getattr(prefix_decode, "paged_gqa_decode_prefix_" + dtype), backend="hip", constexprs=dict(HEAD_GROUP=group), **options)


def i32(values):
    return torch.tensor(values, dtype=torch.int32)


def case(seed, dtype, prefix, lengths, heads, kv_heads, d, ps, spare=0, size=1.0):
    """q, caches, tables and scale on the CPU; pages are scattered, `spare` more entries than a sequence needs hold no page of its own."""
    g = torch.Generator().manual_seed(seed)
    shared = -(-prefix // ps)
    needs = [-(-n // ps) + spare for n in lengths]
    offsets = [0]
    for n in needs:
        offsets.append(offsets[-1] + n)
    where = torch.randperm(shared + offsets[-1], generator=g).to(torch.int32)
    caches = [torch.randn((max(len(where), 1), ps, kv_heads, d), generator=g).to(TYPES[dtype]) for _ in range(2)]
    q = (torch.randn((len(lengths), heads, d), generator=g) * size).to(TYPES[dtype])
    return q, *caches, where[:shared], i32([prefix]), i32(offsets), where[shared:], i32(lengths), float(torch.tensor(d ** -0.5))


def run(device, dtype, given, **options):
    group = given[0].shape[1] // given[1].shape[2]
    return kernel(dtype, group, **options).run(*(t.to(device) for t in given[:8]), given[8])


def check(device, dtype, given):
    prefix_bar.check(run(device, dtype, given), *prefix_bar.bar(*given, dtype))


CASES = [
    # prefix, own lengths, query heads, key heads, d, page
    (1, [0], 1, 1, 64, 16), (0, [1], 2, 1, 128, 16), (31, [1, 32, 33], 8, 2, 64, 16), (32, [0, 5], 4, 4, 128, 32), (33, [64], 6, 2, 128, 64),
    (129, [1, 200, 0, 77], 32, 8, 128, 64), (500, [300, 31], 16, 2, 64, 1), (77, [90, 3], 20, 4, 128, 8), (100, [41] * 5, 17, 1, 128, 24),
    (260, [7] * 3, 40, 2, 64, 48), (2000, [513, 1, 700], 8, 1, 128, 16), (1021, list(range(0, 70)), 8, 2, 64, 16),
    (700, [20] * 40, 16, 2, 128, 32), (64, [1500, 0, 1025], 12, 4, 128, 64), (4100, [10] * 9, 64, 4, 64, 64), (300, [3000], 5, 5, 128, 7),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("prefix,lengths,heads,kv_heads,d,ps", CASES)
def test_matches_plain_form(device, dtype, prefix, lengths, heads, kv_heads, d, ps):
    announce("decode behind a prefix", dtype, prefix, len(lengths), heads, kv_heads, d, ps)
    check(device, dtype, case(prefix + heads, dtype, prefix, lengths, heads, kv_heads, d, ps))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("size", [0.0, 20.0])
def test_flat_and_sharp_weights(device, dtype, size):
    """Equal weights, and weights of which one counts for all: peaks that rise along the walk and apart in its parts."""
    announce("decode behind a prefix, weights", dtype, size)
    check(device, dtype, case(3, dtype, 900, [40, 0, 300], 8, 2, 128, 16, size=size))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("size", [0.0, 1.0, 20.0])
@pytest.mark.parametrize("prefix,lengths,heads,kv_heads,d,ps", [
    (300, [9] * 40, 16, 2, 64, 8), (200, [5, 0] * 15, 8, 1, 128, 20), (270, [33] * 20, 8, 1, 64, 32), (600, [50, 1] * 10, 32, 4, 128, 16)])
def test_two_tiles_of_rows(device, dtype, size, prefix, lengths, heads, kv_heads, d, ps):
    """So many query rows for a key head that a wave takes two tiles of them, whose peaks rise apart from each other."""
    announce("decode behind a prefix, two tiles", dtype, size, prefix, len(lengths), d, ps)
    check(device, dtype, case(6, dtype, prefix, lengths, heads, kv_heads, d, ps, size=size))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("bits", [10, 20, 30])
def test_one_key_outweighs(device, dtype, bits):
    """The first key outweighs every other by 2^bits and has a value of 0, so the output is what the others add."""
    announce("decode behind a prefix, outweighed", dtype, bits)
    given = list(case(4, dtype, 200, [50], 4, 2, 64, 16))
    q, keys, values = given[:3]
    direction = torch.where(torch.arange(64) % 3 == 0, -1.0, 1.0)
    q[:] = direction
    keys[:] = (torch.randint(-1, 2, keys.shape, generator=torch.Generator().manual_seed(1)) / 64).to(keys.dtype)
    first = int(given[3][0])
    keys[first, 0], values[first, 0] = direction.to(keys.dtype), 0
    given[8] = float(torch.tensor(bits / (64 * prefix_bar.LOG2E)))
    check(device, dtype, given)


def test_layouts(device):
    """Pages with their heads one after another, caches inside larger ones, queries of a packed projection, an output with a stride."""
    announce("decode behind a prefix, layouts")
    given = case(5, "bf16", 130, [40, 3, 77], 8, 2, 128, 16)
    want = run(device, "bf16", given)
    on = [t.to(device) for t in given[:8]]
    major = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in on[1:3]]
    inside = [torch.full((c.shape[0] + 2, c.shape[1], 3, 2, 136), float("nan"), dtype=c.dtype, device=device) for c in on[1:3]]
    for whole, c in zip(inside, on[1:3]):
        whole[1:-1, :, 1, :, 8:] = c
    packed = torch.zeros((3, 12, 128), dtype=torch.bfloat16, device=device)
    packed[:, 2:10] = on[0]
    spread = torch.zeros((3, 8, 128, 2), dtype=torch.bfloat16, device=device)
    spread[..., 0] = on[0]
    for caches in (major, [w[1:-1, :, 1, :, 8:] for w in inside]):
        for q in (packed[:, 2:10], spread[..., 0]):
            out = torch.full((3, 8, 2, 129), 7.0, dtype=torch.bfloat16, device=device)
            kernel("bf16", 4)(q, *caches, *on[3:], out[:, :, 1, :128], given[8])
            assert torch.equal(out[:, :, 1, :128], want)
            assert (out[:, :, 0] == 7).all() and (out[:, :, 1, 128] == 7).all()


def test_tables(device):
    """Lengths beyond the pages, below zero, pages that no length reaches, entries outside the cache, no token at all."""
    announce("decode behind a prefix, tables")
    given = list(case(6, "f16", 100, [40, 3, 0, 77], 8, 2, 64, 16, spare=2))
    for name in (1, 2):                                    # what no length reaches does not count, whatever it holds
        reached = torch.zeros(given[name].shape[:2], dtype=torch.bool)
        for pages, first, length in [(given[3], 0, 100)] + [(given[6], given[5][b], given[7][b]) for b in range(4)]:
            at = torch.arange(int(length))
            reached[pages.long()[at // 16 + int(first)], at % 16] = True
        given[name][~reached] = float("nan")
    check(device, "f16", given)
    given = list(case(6, "f16", 100, [40, 3, 0, 77], 8, 2, 64, 16))
    given[4], given[7] = i32([10 ** 9]), i32([10 ** 9, -5, 3, 2 ** 31 - 1])
    check(device, "f16", given)
    given[3][2], given[6][0], given[6][-1] = -7, 10 ** 6, -2 ** 31
    check(device, "f16", given)
    given[4] = i32([-3])
    given[7][:] = 0
    out = run(device, "f16", given)
    assert (out == 0).all()
    empty = case(7, "bf16", 0, [0, 0], 8, 2, 128, 16)
    assert (run(device, "bf16", empty) == 0).all()
    bare = (empty[0], *(c[:0] for c in empty[1:3]), i32([3, 1]), i32([20]), i32([0, 1, 1]), i32([5]), i32([9, 9]), empty[8])
    assert (run(device, "bf16", bare) == 0).all()
    none = (empty[0][:0], *empty[1:5], i32([0]), i32([]), i32([]), empty[8])
    assert run(device, "bf16", none).shape == (0, 8, 128)


def test_special_values(device):
    """NaN and infinities reach the heads that read them and no other; a row of scores of -inf among others weighs nothing."""
    announce("decode behind a prefix, special values")
    given = list(case(8, "bf16", 100, [40, 3], 8, 2, 128, 16))
    want = run(device, "bf16", given)
    shared, own = int(given[3][1]), int(given[6][given[5][1]])
    values = given[2].clone()
    values[shared, 3, 0, 5] = float("nan")
    got = run(device, "bf16", [*given[:2], values, *given[3:]])
    assert got[:, :4, 5].isnan().all()
    keep = torch.ones(got.shape, dtype=torch.bool, device=device)
    keep[:, :4, 5] = False
    assert torch.equal(got[keep], want[keep])
    values = given[2].clone()
    values[own, 1, 1] = float("inf")
    got = run(device, "bf16", [*given[:2], values, *given[3:]])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1, :4], want[1, :4]) and (got[1, 4:] == float("inf")).all()
    q, keys = given[0].clone(), given[1].clone()
    q[:, :4] = q[:, :4].abs() + 0.5
    keys[given[3].long()[:2], :, 0] = float("-inf")        # the first 32 tokens of the prefix
    check(device, "bf16", [q, keys.nan_to_num(neginf=-3e4), *given[2:]])
    got = run(device, "bf16", [q, keys, *given[2:]])
    with_large = run(device, "bf16", [q, keys.nan_to_num(neginf=-3e4), *given[2:]])
    assert torch.equal(got, with_large)


@pytest.mark.parametrize("d,ps", [(64, 16), (128, 20)])
def test_rows_beyond_32_bits(device, d, ps):
    """Pages far apart, tokens far apart."""
    announce("decode behind a prefix, far rows", d, ps)
    given = case(9, "f16", 40, [21, 3], 4, 2, d, ps)
    want = run(device, "f16", given)
    pages = given[1].shape[0]
    stride = 2 ** 31 // pages // 8 * 8 + 4096
    on = [t.to(device) for t in given[:8]]
    for strides in ((stride, 2 * d, d, 1), (2 * d, pages * 2 * d + 2 ** 27, d, 1)):
        far = []
        for c in on[1:3]:
            size = 1 + sum((n - 1) * s for n, s in zip(c.shape, strides))
            far.append(torch.zeros(size, dtype=c.dtype, device=device).as_strided(c.shape, strides).copy_(c))
        assert torch.equal(kernel("f16", 2).run(on[0], *far, *on[3:], given[8]), want)


def test_captured_steps(device):
    """Captured twice and replayed between eager calls while lengths, pages and queries change; on another stream as well."""
    announce("decode behind a prefix, captured")
    given = case(10, "bf16", 333, [100, 200, 7, 50], 16, 4, 128, 16)
    on = [t.to(device) for t in given[:8]]
    on[3], on[6] = on[3].clone(), on[6].clone()
    one = kernel("bf16", 4)
    call = one.prepare(*on, given[8])
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call.launch()
        graphs.append(graph)
    side = torch.cuda.Stream()
    for step in range(5):
        on[4].fill_(333 - 40 * step)
        on[7].copy_(i32([100 - step, 10 * step, 7, 0 if step == 2 else 50]))
        on[3].copy_(on[3].roll(1))
        on[0].copy_(torch.roll(on[0], 1, 0))
        want = kernel("bf16", 4).run(*on, given[8])
        call.result().zero_()
        if step < 4:
            graphs[step % 2].replay()
        else:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                call.launch()
            torch.cuda.current_stream().wait_stream(side)
        again = one.run(*on, given[8])
        torch.cuda.synchronize()
        assert torch.equal(call.result(), want) and torch.equal(again, want)
        prefix_bar.check(want, *prefix_bar.bar(*(t.cpu() for t in on), given[8], "bf16"))


def test_refusals(device):
    given = [t.to(device) for t in case(1, "f16", 40, [20, 3], 8, 2, 64, 16)[:8]]
    one = kernel("f16", 4)
    with pytest.raises(ValueError, match="HEAD_GROUP"):
        kernel("f16", 2).run(*given, 0.1)
    with pytest.raises(ValueError, match="batch"):
        one.run(*given[:5], given[5][:-1], *given[6:], 0.1)
    with pytest.raises(ValueError, match="one number"):
        one.run(*given[:4], given[4].repeat(2), *given[5:], 0.1)
    with pytest.raises(ValueError, match="aligned"):
        one.run(given[0], torch.zeros((*given[1].shape[:3], 68), dtype=torch.float16, device=device)[..., :64], *given[2:], 0.1)
    with pytest.raises(TypeError):
        one.run(given[0].bfloat16(), *given[1:], 0.1)
    with pytest.raises(intent.CompilationStageError, match="64 or 128"):
        wide = torch.zeros((4, 16, 2, 96), dtype=torch.float16, device=device)
        one.run(torch.zeros((2, 8, 96), dtype=torch.float16, device=device), wide, wide.clone(), *given[3:], 0.1)
    with pytest.raises(intent.CompilationStageError, match="HEAD_GROUP"):
        kernel("f16", 0).run(*given, 0.1)
    with pytest.raises(intent.CompilationStageError, match="workspace"):
        kernel("f16", 4, backend_options={"workspace": "static"}).run(*given, 0.1)
    one.run(*given, 0.1)
