"""paged_gqa_decode_mx against its 64-bit form.

Bar. A score in the exponent of two is an f32 sum of D exact products, scaled: off by at most (D + 2) * 2^-24 of the sum of
their magnitudes, which is bounded from the inputs; a weight is off by that share (times ln 2), once in the numerator and once
in the denominator. The weights' two parts leave 2^-14 (bf16) of them; the f32 sums run in chains of at most 2^7 steps of 8
keys, 2^-14 of the sum of weight * |value| with the joins. Then half a step of the output type."""
import pytest
import torch

import intent_amd as intent
from intent_amd.examples.kernels.streaming import mx_cache
from tests import plain64
from tests.gpu_util import announce
from tests.test_gpu_mx_cache import cache, i32, tables

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def kernel(dtype, group):
    return intent.jit(getattr(mx_cache, "paged_gqa_decode_mx_" + dtype), backend="hip", constexprs={"HEAD_GROUP": group})


def filled(generator, pages, page, heads, d, head_major, device, fill=0x7F):
    """A cache whose places hold random rows, and what they stand for; `fill` (NaN) is what other places hold."""
    held = cache(pages, page, heads, d, head_major, device, fill)
    rows = torch.randn((pages, page, heads, d), generator=generator) * torch.exp2(torch.randint(-2, 3, (pages, page, heads, 1), generator=generator))
    elements, powers = plain64.quantise(rows)
    held[0].view(torch.uint8).copy_(elements.float().to(torch.float8_e4m3fn).view(torch.uint8))
    held[1].copy_(powers.to(torch.uint8))
    return held, plain64.dequantise(elements, powers)


def poison(held, offsets, indices, lengths):
    """NaN in every place without a token."""
    pages, page = held[0].shape[:2]
    free = torch.ones((pages, page), dtype=torch.bool)
    for s, n in enumerate(lengths):
        for p in range(min(n, (offsets[s + 1] - offsets[s]) * page)):
            free[int(indices[offsets[s] + p // page]), p % page] = False
    for at in free.nonzero().tolist():
        held[0][tuple(at)].view(torch.uint8).fill_(0x7F)
        held[1][tuple(at)].fill_(255)


def check(out, q, keys, values, offsets, indices, lengths, scale, dtype):
    want, size = plain64.decode(q.double(), keys, values, offsets, indices, lengths, scale)
    got = out.double().cpu()
    assert not got.isnan().any()
    # the largest sum of magnitudes of a score, in the exponent of two
    magnitude = float(q.double().abs().amax() * keys.abs().nan_to_num().amax()) * q.shape[2] * scale * 1.4427
    units = 2 * (q.shape[2] + 2) * 2.0 ** -24 * magnitude + 2.0 ** -14 + 2.0 ** -14
    bound = HALF_STEP[dtype] * want.abs() + units * size + 2.0 ** -25
    worst = (got - want).abs() - bound
    assert (worst <= 0).all(), f"off by {(got - want).abs().flatten()[worst.argmax()]} of {want.flatten()[worst.argmax()]}"


CASES = [([1], 1, 1, 64, 16, True), ([0, 1, 15, 16, 17], 4, 2, 64, 16, False), ([31, 32, 33, 0, 0], 8, 1, 128, 16, True),
         ([129, 127, 128], 1, 4, 128, 64, True), ([700, 3, 1290], 4, 2, 128, 32, False), ([65, 200], 16, 1, 96, 64, True),
         ([300, 41], 17, 1, 128, 64, True), ([90], 40, 2, 64, 16, False), ([513, 1], 3, 5, 192, 48, True),
         ([260, 77], 2, 2, 256, 64, False), ([100, 7, 33], 4, 2, 128, 1, True), ([100, 7, 33], 20, 1, 64, 7, False),
         ([95, 0, 130], 4, 2, 96, 24, True), ([64, 31], 5, 1, 256, 10, True), ([0, 0], 4, 1, 128, 16, True),
         ([4000, 1, 2500, 64], 4, 1, 128, 64, True)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lengths,group,heads,d,page,head_major", CASES)
def test_matches_plain_form(device, dtype, lengths, group, heads, d, page, head_major):
    """Lengths around a tile, a step and a job, groups around a tile of heads, pages that a tile of keys crosses; places
    without a token hold NaN."""
    announce("mx decode", dtype, lengths, group, heads, d, page, head_major)
    g = torch.Generator().manual_seed(sum(lengths) + group + d)
    pages, offsets, indices = tables(lengths, page, g)
    keys, plain_keys = filled(g, pages, page, heads, d, head_major, device)
    values, plain_values = filled(g, pages, page, heads, d, head_major, device)
    for held in (keys, values):
        poison(held, offsets, indices, lengths)
    q = torch.randn((len(lengths), heads * group, d), generator=g).to(TYPES[dtype])
    scale = d ** -0.5
    out = kernel(dtype, group).run(q.to(device), *keys, *values, i32(offsets, device), indices.to(device), i32(lengths, device), scale)
    check(out, q, plain_keys, plain_values, offsets, indices, lengths, scale, dtype)


def test_reserved_pages_and_lengths_past_them(device):
    """Pages reserved ahead of a sequence are not read; a length beyond its pages ends with them; a page outside the cache has
    no token; a negative length is none; offsets may start behind 0."""
    announce("mx decode with reserved and missing pages")
    g = torch.Generator().manual_seed(11)
    keys, plain_keys = filled(g, 12, 16, 2, 64, True, device)
    values, plain_values = filled(g, 12, 16, 2, 64, True, device)
    offsets, indices = [1, 5, 6, 9, 10, 12], torch.tensor([9, 3, 7, 11, 0, 2, 4, 99, 6, 5, -1, 8], dtype=torch.int32)
    lengths = [18, 1000, 48, -5, 30]
    q = torch.randn((5, 8, 64), generator=g).half()
    out = kernel("f16", 4).run(q.to(device), *keys, *values, i32(offsets, device), indices.to(device), i32(lengths, device), 0.125)
    check(out, q, plain_keys, plain_values, offsets, indices, lengths, 0.125, "f16")
    assert (out[3] == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page,held", [(16, [3, 2, 4]), (7, [3, 2, 4]), (16, [400, 90, 3]), (5, [600, 700, 3])])
def test_sequences_whose_pages_are_all_outside(device, dtype, page, held):
    """A sequence that has pages, but none in the cache, gives 0, as do jobs of a longer one; its neighbours are not touched."""
    announce("mx decode with no page inside", dtype, page, held)
    g = torch.Generator().manual_seed(sum(held) + page)
    keys, plain_keys = filled(g, 40, page, 2, 64, True, device)
    values, plain_values = filled(g, 40, page, 2, 64, True, device)
    offsets = [0, held[0], held[0] + held[1], sum(held)]
    indices = torch.randint(0, 40, (sum(held),), generator=g, dtype=torch.int32)
    indices[offsets[0]:offsets[1]] = torch.where(torch.arange(held[0]) % 2 == 0, -1, 40).int()
    indices[offsets[1]:offsets[1] + held[1] // 2] = 1 << 30
    lengths = [n * page for n in held]
    q = torch.randn((3, 8, 64), generator=g).to(TYPES[dtype])
    out = kernel(dtype, 4).run(q.to(device), *keys, *values, i32(offsets, device), indices.to(device), i32(lengths, device), 0.125)
    assert (out[0] == 0).all()
    check(out, q, plain_keys, plain_values, offsets, indices, lengths, 0.125, dtype)


def test_caches_without_a_page(device):
    """No page, pages of no token and an empty table give 0, whatever the lengths say."""
    announce("mx decode without pages")
    q = torch.randn((3, 8, 64), device=device).half()
    for pages, ps, positions in ((0, 16, 4000), (0, 16, 4), (4, 0, 4), (2, 16, 0)):
        held = [torch.zeros((pages, ps, 2, w), dtype=torch.uint8, device=device) for w in (64, 2, 64, 2)]
        held[0], held[2] = held[0].view(torch.float8_e4m3fn), held[2].view(torch.float8_e4m3fn)
        out = torch.full((3, 8, 64), 7.0, dtype=torch.float16, device=device)
        offsets = i32([0, positions // 2, positions // 2, positions], device)
        kernel("f16", 4)(q, *held, offsets, torch.zeros(positions, dtype=torch.int32, device=device), i32([50, 3, 9], device), out, 1.0)
        assert (out == 0).all()


def test_rising_scores_and_large_ones(device):
    """Scores that rise along the sequence raise the running maximum again and again; scores of hundreds leave one key."""
    announce("mx decode with rising scores")
    g = torch.Generator().manual_seed(12)
    for factor in (0.01, 1.0, 40.0):
        keys, plain_keys = filled(g, 16, 64, 1, 128, True, device)
        values, plain_values = filled(g, 16, 64, 1, 128, True, device)
        direction = torch.randn(128, generator=g)
        direction /= direction.norm()
        rows = direction * torch.arange(1024)[:, None] * factor / 64
        elements, powers = plain64.quantise(rows)
        keys[0].transpose(1, 2).view(torch.uint8).copy_(elements.float().to(torch.float8_e4m3fn).view(torch.uint8).view(16, 1, 64, 128))
        keys[1].transpose(1, 2).copy_(powers.to(torch.uint8).view(16, 1, 64, 4))
        plain_keys = plain64.dequantise(elements, powers).view(16, 64, 1, 128)
        q = (direction + 0.05 * torch.randn((1, 4, 128), generator=g)).half()
        order = torch.arange(16, dtype=torch.int32)
        out = kernel("f16", 4).run(q.to(device), *keys, *values, i32([0, 16], device), order.to(device), i32([1000], device), 1.0)
        check(out, q, plain_keys, plain_values, [0, 16], order, [1000], 1.0, "f16")


def test_special_values(device):
    """A NaN key or value, and an infinite score, reach the heads that see them and no others."""
    announce("mx decode with NaN")
    g = torch.Generator().manual_seed(13)
    keys, _ = filled(g, 4, 16, 2, 64, True, device)
    values, _ = filled(g, 4, 16, 2, 64, True, device)
    q = torch.randn((2, 4, 64), generator=g).half().to(device)
    table = (i32([0, 2, 4], device), i32([0, 1, 2, 3], device), i32([20, 32], device))
    run = lambda: kernel("f16", 2).run(q, *keys, *values, *table, 0.125)  # noqa: E731
    want = run()
    keys[0].view(torch.uint8)[0, 3, 1, 5] = 0x7F
    got = run()
    assert got[0, 2:].isnan().all() and torch.equal(got[0, :2], want[0, :2]) and torch.equal(got[1], want[1])
    keys[0].view(torch.uint8)[0, 3, 1, 5] = 0x30
    values[1][2, 0, 0, 0] = 255
    got = run()
    assert got[1, :2, :32].isnan().all() and not got[1, :2, 32:].isnan().any() and torch.equal(got[1, 2:], want[1, 2:])


def test_layouts_streams_and_graphs(device):
    """Queries and outputs of odd layouts, a launch on another stream than the one it was prepared on, and two captured graphs
    whose lengths change between replays, against fresh calls."""
    announce("mx decode layouts, streams, graphs")
    g = torch.Generator().manual_seed(14)
    lengths = i32([3000, 40, 1], device)
    offsets, order = i32([0, 60, 120, 180], device), torch.randperm(180, generator=g).to(torch.int32).to(device)
    keys, _ = filled(g, 180, 64, 2, 128, False, device)
    values, _ = filled(g, 180, 64, 2, 128, False, device)
    q = torch.randn((3, 8, 128), generator=g).half().to(device)
    run = kernel("f16", 4)
    want = run.run(q, *keys, *values, offsets, order, lengths, 0.09)
    odd = torch.zeros((3, 8, 131), dtype=torch.float16, device=device)
    odd[..., 1:129] = q
    out = torch.zeros((3, 8, 128, 2), dtype=torch.float16, device=device)
    run(odd[..., 1:129], *keys, *values, offsets, order, lengths, out[..., 0], 0.09)
    assert torch.equal(out[..., 0], want) and not out[..., 1].any()
    call = run.prepare(q, *keys, *values, offsets, order, lengths, 0.09)
    assert dict(call._launch.configuration)["workspace_bytes"] > 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call.launch()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(call.result(), want)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call.launch()
        graphs.append(graph)
    for step in range(4):
        lengths.copy_(i32([3000 - 700 * step, 40 + 900 * step, step], device))
        call.result().zero_()
        graphs[step % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(call.result(), run.run(q, *keys, *values, offsets, order, lengths, 0.09))


def test_refusals(device):
    g = torch.Generator().manual_seed(15)
    keys, _ = filled(g, 2, 16, 2, 64, True, device)
    values, _ = filled(g, 2, 16, 2, 64, True, device)
    q = torch.zeros((1, 8, 64), dtype=torch.float16, device=device)
    table = (i32([0, 2], device), i32([0, 1], device), i32([20], device))
    kernel("f16", 4).run(q, *keys, *values, *table, 1.0)
    with pytest.raises(ValueError, match="HEAD_GROUP"):
        kernel("f16", 2).run(q, *keys, *values, *table, 1.0)
    with pytest.raises(intent.CompilationStageError, match="HEAD_GROUP"):
        kernel("f16", 0).run(q, *keys, *values, *table, 1.0)
    with pytest.raises(ValueError, match="page_offsets"):
        kernel("f16", 4).run(q, *keys, *values, i32([0, 1, 2], device), *table[1:], 1.0)
    with pytest.raises(TypeError):
        kernel("bf16", 4).run(q, *keys, *values, *table, 1.0)
    with pytest.raises(ValueError):
        kernel("f16", 4).run(q, keys[0], keys[1], *cache(2, 16, 2, 128, True, device), *table, 1.0)
    with pytest.raises(intent.CompilationStageError, match="head widths"):
        wide = cache(2, 16, 2, 32, True, device)
        kernel("f16", 4).run(q[..., :32], *wide, *wide, *table, 1.0)
    with pytest.raises(ValueError, match="multiples of 16"):
        odd = torch.zeros((2, 16, 2, 72), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)[..., :64]
        kernel("f16", 4).run(q, odd, keys[1], *values, *table, 1.0)
    static = intent.jit(mx_cache.paged_gqa_decode_mx_f16, backend="hip", constexprs={"HEAD_GROUP": 4},
                        backend_options={"workspace": "static"})
    static.run(q, *keys, *values, *table, 1.0)                            # one job: no workspace
    with pytest.raises(intent.CompilationStageError, match="workspace"):
        static.run(q, *keys, *values, table[0], torch.zeros(4000, dtype=torch.int32, device=device), table[2], 1.0)


@pytest.mark.parametrize("batch,positions", [(200, 900), (3, 3000), (70, 65)])
def test_many_sequences_and_jobs(device, batch, positions):
    """More sequences than a wave has lanes, and long page lists cut into many jobs: each job finds its sequence, also behind
    sequences without a page; every row is joined from its own states."""
    announce("mx decode many sequences", batch, positions)
    g = torch.Generator().manual_seed(batch)
    ends = torch.randint(0, positions + 1, (batch - 1,), generator=g).sort().values
    offsets = [0, *ends.tolist(), positions]
    counts = [b - a for a, b in zip(offsets, offsets[1:])]
    lengths = [max(0, n * 16 - int(torch.randint(0, 16, (1,), generator=g))) for n in counts]
    pages = 40                                                     # shared by the sequences, again and again
    indices = torch.randint(0, pages, (positions,), generator=g).to(torch.int32)
    keys, plain_keys = filled(g, pages, 16, 1, 64, True, device)
    values, plain_values = filled(g, pages, 16, 1, 64, True, device)
    q = torch.randn((batch, 2, 64), generator=g).half()
    out = kernel("f16", 2).run(q.to(device), *keys, *values, i32(offsets, device), indices.to(device), i32(lengths, device), 0.125)
    check(out, q, plain_keys, plain_values, offsets, indices, lengths, 0.125, "f16")


def test_scale_of_either_sign_and_none(device):
    announce("mx decode scales")
    g = torch.Generator().manual_seed(16)
    keys, plain_keys = filled(g, 4, 16, 1, 64, True, device)
    values, plain_values = filled(g, 4, 16, 1, 64, True, device)
    poison(keys, [0, 4], torch.arange(4), [50])
    poison(values, [0, 4], torch.arange(4), [50])
    q = torch.randn((1, 3, 64), generator=g).half()
    table = (i32([0, 4], device), i32([0, 1, 2, 3], device), i32([50], device))
    for scale in (-0.2, 0.0):
        out = kernel("f16", 3).run(q.to(device), *keys, *values, *table, scale)
        want, size = plain64.decode(q, plain_keys, plain_values, [0, 4], [0, 1, 2, 3], [50], scale)
        assert not out.isnan().any()
        assert ((out.double().cpu() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -13 * size).all()


def test_offsets_beyond_32_bits(device):
    """Pages behind the first 4 GiB of a cache, and a token stride whose lane offsets would pass 32 bits."""
    announce("mx decode beyond 32 bits")
    g = torch.Generator().manual_seed(31)
    near, plain_near = filled(g, 6, 16, 1, 64, False, device)
    values, plain_values = filled(g, 6, 16, 1, 64, False, device)
    pages = 2 ** 32 // (16 * 64) + 7
    q = torch.randn((2, 4, 64), generator=g).half()
    offsets, indices, lengths = [0, 4, 6], torch.tensor([5, 0, 3, 1, 2, 4], dtype=torch.int32), [61, 18]
    far = torch.where(indices % 2 == 0, indices, indices + pages - 6).int()
    caches = []
    for elements, exponents in (near, values):
        wide = torch.zeros((pages, 16, 1, 64), dtype=torch.uint8, device=device)
        powers = torch.zeros((pages, 16, 1, 2), dtype=torch.uint8, device=device)
        assert wide.numel() > 2 ** 32
        for a, b in zip(indices.tolist(), far.tolist()):
            wide[b], powers[b] = elements[a].view(torch.uint8), exponents[a]
        caches += [wide.view(torch.float8_e4m3fn), powers]
    run = lambda held, at: kernel("f16", 4).run(q.to(device), *held, i32(offsets, device), at.to(device), i32(lengths, device), 0.125)  # noqa: E731
    out = run(caches, far)
    check(out, q, plain_near, plain_values, offsets, indices, lengths, 0.125, "f16")
    del caches, wide, powers
    strided = []
    for elements, exponents in (near, values):
        store = torch.zeros(15 * 2 ** 26 + 6 * 64, dtype=torch.uint8, device=device)
        view = store.as_strided((6, 16, 1, 64), (64, 2 ** 26, 64, 1))
        view.copy_(elements.view(torch.uint8))
        strided += [view.view(torch.float8_e4m3fn), exponents]
    check(run(strided, indices), q, plain_near, plain_values, offsets, indices, lengths, 0.125, "f16")
