"""paged_cache_append and paged_cache_read against their 64-bit forms, exactly: scaling by a power of two is exact, so the
elements, the exponents and the values read back (one rounding to the row type) have one right answer each."""
import pytest
import torch

import intent_amd as intent
from intent_amd.examples.kernels.streaming import mx_cache
from tests import plain64
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def kernel(name):
    return intent.jit(getattr(mx_cache, name), backend="hip")


def i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def tables(lengths, page, generator, spare=3):
    """(pages, page_offsets, page_indices): every sequence's pages scattered over the cache, `spare` pages nobody's."""
    offsets = [0]
    for n in lengths:
        offsets.append(offsets[-1] + -(-n // page))
    order = torch.randperm(offsets[-1] + spare, generator=generator)
    return offsets[-1] + spare, offsets, order[:offsets[-1]].to(torch.int32)


def cache(pages, page, heads, dim, head_major, device, fill=0x55):
    shape = (pages, heads, page) if head_major else (pages, page, heads)
    elements = torch.full((*shape, dim), fill, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    exponents = torch.full((*shape, dim // 32), 121, dtype=torch.uint8, device=device)
    return (elements.transpose(1, 2), exponents.transpose(1, 2)) if head_major else (elements, exponents)


def bits(elements):
    return elements.contiguous().view(torch.uint8).cpu()


def expected(before, rows, slots):
    """Elements (as floats) and exponents of a cache after `rows` went to `slots` (None: nowhere)."""
    elements, exponents = before[0].contiguous().float().double().cpu(), before[1].contiguous().int().cpu()
    held, powers = plain64.quantise(rows)
    for i, slot in enumerate(slots):
        if slot is not None:
            elements[slot], exponents[slot] = held[i], powers[i]
    return elements, exponents


CASES = [([1], [1], 1, 1, 32, 32, True), ([5, 0, 17, 64], [5, 0, 1, 64], 16, 2, 64, 64, False),
         ([5, 0, 17, 64], [1, 0, 17, 3], 16, 2, 64, 64, True), ([130, 1, 63], [130, 1, 63], 64, 8, 128, 128, True),
         ([33, 70], [33, 8], 7, 3, 96, 32, False), ([300], [290], 32, 5, 256, 128, True), ([9, 9, 9], [9, 9, 9], 1, 1, 32, 64, False)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lengths,new,page,heads,d,dv,head_major", CASES)
def test_append_then_read(device, dtype, lengths, new, page, heads, d, dv, head_major):
    """New tokens go to their slots and nowhere else, with rows behind the last sequence; what is read back is what they
    stand for, and rows behind the last sequence keep what they held."""
    announce("cache append and read", dtype, lengths, new, page, heads, d, dv, head_major)
    g = torch.Generator().manual_seed(sum(lengths) + d)
    pages, offsets, indices = tables(lengths, page, g)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    padded = cu[-1] + 2
    scale = torch.exp2(torch.randint(-6, 4, (padded, heads, 1), generator=g))       # blocks of different sizes
    k = (torch.randn((padded, heads, d), generator=g) * scale).to(TYPES[dtype])
    v = (torch.randn((padded, heads, dv), generator=g) * scale).to(TYPES[dtype])
    keys, values = (cache(pages, page, heads, w, head_major, device) for w in (d, dv))
    before = [(c[0].clone(), c[1].clone()) for c in (keys, values)]
    slots = [(int(indices[offsets[s] + p // page]), p % page) for s, n in enumerate(lengths)
             for p in range(n - new[s], n)] + [None, None]
    rows = torch.cat((k, v), -1).to(device)                                          # strided slices of one tensor
    kernel("paged_cache_append_" + dtype).run(rows[..., :d], rows[..., d:], *keys, *values, i32(cu, device), i32(offsets, device),
                                              indices.to(device), i32(lengths, device))
    for held, old, x in zip((keys, values), before, (k, v)):
        want, powers = expected(old, x, slots)
        assert torch.equal(held[0].contiguous().float().double().cpu(), want)
        assert torch.equal(held[1].contiguous().int().cpu(), powers)

    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    outs = [torch.full((ends[-1] + 2, heads, w), 7.0, dtype=TYPES[dtype], device=device) for w in (d, dv)]
    kernel("paged_cache_read_" + dtype)(*keys, *values, i32(ends, device), i32(offsets, device), indices.to(device), *outs)
    for out, held in zip(outs, (keys, values)):
        whole = plain64.dequantise(held[0].contiguous().float().cpu(), held[1].contiguous().cpu()).to(TYPES[dtype])
        want = torch.stack([whole[int(indices[offsets[s] + p // page]), p % page] for s, n in enumerate(lengths) for p in range(n)])
        assert torch.equal(out[:-2].cpu(), want)
        assert (out[-2:] == 7).all()


@pytest.mark.parametrize("sequences", [1, 63, 64, 65, 130, 4096, 5000])
def test_many_sequences(device, sequences):
    """One new token for each of many sequences (some have none), found among the offsets by every wave."""
    announce("cache append of many sequences", sequences)
    g = torch.Generator().manual_seed(sequences)
    new = torch.randint(0, 3, (sequences,), generator=g)
    cu = torch.cat((torch.zeros(1, dtype=torch.int64), new.cumsum(0))).to(torch.int32)
    lengths = (new + torch.randint(0, 2, (sequences,), generator=g)).to(torch.int32)
    offsets = torch.arange(sequences + 1, dtype=torch.int32)                         # a page of 4 for each
    keys, values = (cache(sequences, 4, 1, 32, True, device) for _ in range(2))
    k = torch.randn((int(cu[-1]), 1, 32), generator=g).half()
    kernel("paged_cache_append_f16").run(k.to(device), k.to(device), *keys, *values, cu.to(device), offsets.to(device),
                                         offsets[:-1].to(device), lengths.to(device))
    held, powers = plain64.quantise(k)
    want = torch.full((sequences, 4, 1, 32), 0x55, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    sequence = torch.repeat_interleave(torch.arange(sequences), new)
    place = torch.arange(int(cu[-1])) - cu[:-1].long()[sequence] + (lengths.long() - new)[sequence]
    want[sequence, place] = held
    for elements, _ in (keys, values):
        assert torch.equal(elements.contiguous().float().double().cpu(), want)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_every_rounding(device, dtype):
    """Blocks whose largest value sits at, just below and just above 448 * 2^e for every e of the type, values at and next to
    every half between elements, subnormals, zeros, NaN and infinities."""
    announce("cache roundings", dtype)
    kind = TYPES[dtype]
    sizes = []
    low, high = (-24, 15) if dtype == "f16" else (-133, 127)
    for e in range(low, high + 1):
        for m in (1.0, 1.0625, 1.71875, 1.75, 1.7578125, 1.9921875):
            sizes.append(m * 2.0 ** e)
    sizes = torch.tensor(sizes, dtype=torch.float64).to(kind)
    elements = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    elements = elements[elements.isfinite()].sort().values
    halves = (elements[1:] + elements[:-1]) / 2
    near = torch.cat((halves, halves * (1 + 2.0 ** -7), halves * (1 - 2.0 ** -7), elements))
    g = torch.Generator().manual_seed(1)
    rows = torch.empty((len(sizes), 32), dtype=torch.float64)
    for i, size in enumerate(sizes.double()):
        exponent = torch.frexp(size)[1] - 9
        rows[i] = torch.ldexp(near[torch.randint(0, len(near), (32,), generator=g)], exponent.expand(32))
        rows[i].clamp_(-float(size), float(size))
        rows[i, i % 32] = size if i % 2 else -size
    special = torch.zeros((4, 32), dtype=torch.float64)
    special[0, 3], special[1, 5], special[1, 6] = float("nan"), float("inf"), -float("inf")
    special[1, 7], special[2] = 3.0, float("inf")
    rows = torch.cat((rows, special)).to(kind)[:, None]
    count = rows.shape[0]
    keys, values = (cache(count, 1, 1, 32, True, device) for _ in range(2))
    kernel("paged_cache_append_" + dtype).run(rows.to(device), rows.to(device), *keys, *values, i32([0, count], device),
                                              i32([0, count], device), torch.arange(count, dtype=torch.int32, device=device),
                                              i32([count], device))
    want, powers = plain64.quantise(rows)
    for elements, exponents in (keys, values):
        got = elements.contiguous().float().double().cpu()[:, 0]
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
        assert torch.equal(exponents.contiguous().int().cpu()[:, 0], powers)
    assert int((want.isnan()).sum()) == 35


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_read_every_element_and_exponent(device, dtype):
    """All 256 elements at all 256 exponents: the value rounded to the type, infinity beyond it, NaN at exponent 255."""
    announce("cache read of every element", dtype)
    elements = torch.arange(256, dtype=torch.uint8).repeat(256, 1)
    exponents = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 8)
    wide = elements.view(256, 1, 1, 256).to(device).view(torch.float8_e4m3fn), exponents.view(256, 1, 1, 8).to(device)
    order = torch.arange(256, dtype=torch.int32, device=device)
    outs = [torch.empty((256, 1, 256), dtype=TYPES[dtype], device=device) for _ in range(2)]
    kernel("paged_cache_read_" + dtype)(*wide, *wide, i32([0, 256], device), i32([0, 256], device), order, *outs)
    want = plain64.dequantise(elements.view(torch.float8_e4m3fn).double(), exponents).to(TYPES[dtype])[:, None]
    for out in outs:
        got = out.cpu()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_bad_tables_leave_the_cache_alone(device):
    """Pages outside the cache, positions before 0 and behind a sequence's pages, offsets outside the index array and rows
    before the first sequence: such rows are not written, and read as 0 (or stay, where no sequence has them)."""
    announce("cache with bad tables")
    g = torch.Generator().manual_seed(2)
    k = torch.randn((8, 1, 32), generator=g).half().to(device)

    def append(cu, offsets, indices, lengths):
        keys, values = (cache(4, 2, 1, 32, True, device) for _ in range(2))
        kernel("paged_cache_append_f16").run(k, k, *keys, *values, i32(cu, device), i32(offsets, device), i32(indices, device),
                                             i32(lengths, device))
        written = (bits(keys[0]) != 0x55).any(-1)[..., 0]
        assert torch.equal(written, (bits(values[0]) != 0x55).any(-1)[..., 0])
        return sorted((p, o) for p, o in written.nonzero().tolist())

    assert append([0, 3], [0, 2], [2, 0], [3]) == [(0, 0), (2, 0), (2, 1)]
    assert append([0, 3], [0, 2], [2, 4], [3]) == [(2, 0), (2, 1)]             # page 4 of 4
    assert append([0, 3], [0, 2], [-1, 0], [3]) == [(0, 0)]
    assert append([0, 3], [0, 2], [2, 0], [2]) == [(2, 0), (2, 1)]             # 3 new tokens of 2: the first has position -1
    assert append([0, 3], [0, 1], [2, 0], [3]) == [(2, 0), (2, 1)]             # position 2 is behind the only page
    assert append([0, 3], [1, 9], [2, 0], [3]) == [(0, 0), (0, 1)]             # offsets past the index array
    assert append([0, 3], [-1, 1], [2, 0], [3]) == []
    assert append([2, 3], [0, 2], [2, 0], [1]) == [(2, 0)]                     # rows 0 and 1 are nobody's
    assert append([0, 0], [0, 2], [2, 0], [3]) == []
    keys, values = (cache(4, 2, 1, 32, True, device) for _ in range(2))
    outs = [torch.full((6, 1, 32), 7.0, dtype=torch.float16, device=device) for _ in range(2)]
    kernel("paged_cache_read_f16")(*keys, *values, i32([1, 4], device), i32([0, 1], device), i32([9], device), *outs)
    assert (outs[0][0] == 7).all() and (outs[0][1:4] == 0).all() and (outs[0][4:] == 7).all()


def test_layouts_of_rows(device):
    """Rows with an odd start, odd strides or an inner stride of 2 are staged; what they write and read is the same."""
    announce("cache rows of odd layouts")
    g = torch.Generator().manual_seed(3)
    k = torch.randn((5, 2, 64), generator=g).half().to(device)
    tail = (i32([0, 5], device), i32([0, 2], device), i32([1, 0], device))
    want = [cache(2, 4, 2, 64, False, device) for _ in range(2)]
    kernel("paged_cache_append_f16").run(k, k, *want[0], *want[1], *tail, i32([5], device))
    odd = torch.zeros((5, 2, 67), dtype=torch.float16, device=device)
    odd[..., 1:65] = k
    inner = torch.zeros((5, 2, 64, 2), dtype=torch.float16, device=device)
    inner[..., 0] = k
    got = [cache(2, 4, 2, 64, False, device) for _ in range(2)]
    kernel("paged_cache_append_f16").run(odd[..., 1:65], inner[..., 0], *got[0], *got[1], *tail, i32([5], device))
    for a, b in zip(want, got):
        assert torch.equal(bits(a[0]), bits(b[0])) and torch.equal(a[1], b[1])
    outs = [torch.empty((7, 2, 64), dtype=torch.float16, device=device) for _ in range(2)]
    kernel("paged_cache_read_f16")(*want[0], *want[1], *tail, *outs)
    odd.fill_(3.0), inner.fill_(3.0)
    wide = [torch.full((7, 2, 67), 3.0, dtype=torch.float16, device=device), torch.full((7, 2, 64, 2), 3.0, dtype=torch.float16, device=device)]
    kernel("paged_cache_read_f16")(*want[0], *want[1], *tail, wide[0][..., 1:65], wide[1][..., 0])
    assert torch.equal(wide[0][:5, :, 1:65], outs[0][:5]) and torch.equal(wide[1][:5, ..., 0], outs[1][:5])
    assert (wide[0][5:] == 3).all() and (wide[1][5:] == 3).all() and (wide[0][..., 65:] == 3).all()


def test_refusals(device):
    keys, values = (cache(4, 2, 1, 64, False, device) for _ in range(2))
    k = torch.zeros((3, 1, 64), dtype=torch.float16, device=device)
    table = (i32([0, 3], device), i32([0, 2], device), i32([2, 0], device), i32([3], device))
    append = kernel("paged_cache_append_f16")
    append.run(k, k, *keys, *values, *table)
    with pytest.raises(TypeError):
        append.run(k.bfloat16(), k, *keys, *values, *table)
    with pytest.raises(ValueError, match="blocks of 32"):
        append.run(k, k, keys[0], keys[1][..., :1], *values, *table)
    narrow = cache(4, 2, 1, 64, False, device)[0][..., :48]
    with pytest.raises(ValueError, match="blocks of 32"):
        append.run(k[..., :48], k, narrow, keys[1], *values, *table)
    with pytest.raises(ValueError, match="multiples of 16"):
        wide = torch.zeros((4, 2, 1, 72), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        append.run(k, k, wide[..., :64], keys[1], *values, *table)
    with pytest.raises(ValueError, match="unit inner stride"):
        append.run(k, k, keys[0], torch.zeros((4, 2, 1, 2, 2), dtype=torch.uint8, device=device)[..., 0], *values, *table)
    with pytest.raises(ValueError, match="overlap"):
        append.run(k, k, *keys, *keys, *table)
    with pytest.raises(ValueError):
        append.run(k, k, *keys, *values, *table[:3], i32([3, 3], device))
    with pytest.raises(NotImplementedError, match="explicit output buffers"):
        kernel("paged_cache_read_f16").run(*keys, *values, *table[:3])


def test_offsets_beyond_32_bits(device):
    """A cache of more than 2^32 bytes: its last page is written and read where it is."""
    announce("cache of more than 2^32 bytes")
    pages, page, heads, d = 2049, 64, 128, 256                    # 4.3 GB of keys; the values are one block wide
    key_elements = torch.zeros((pages, heads, page, d), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn).transpose(1, 2)
    key_exponents = torch.zeros((pages, heads, page, d // 32), dtype=torch.uint8, device=device).transpose(1, 2)
    values = cache(pages, page, heads, 32, True, device)
    assert key_elements.numel() > 2 ** 32
    g = torch.Generator().manual_seed(4)
    k, v = torch.randn((1, heads, d), generator=g).half(), torch.randn((1, heads, 32), generator=g).half()
    tables_ = (i32([0, 1], device), i32([0, 1], device), i32([pages - 1], device))
    kernel("paged_cache_append_f16").run(k.to(device), v.to(device), key_elements, key_exponents, *values, *tables_, i32([64], device))
    held, powers = plain64.quantise(k)
    assert torch.equal(key_elements[-1, -1].float().double().cpu(), held[0])
    assert torch.equal(key_exponents[-1, -1].int().cpu(), powers[0])
    flat = key_elements.transpose(1, 2).view(torch.uint8)
    assert not flat[:-1].any() and int(flat[-1, :, :-1].sum()) == 0
    outs = [torch.empty((64, heads, w), dtype=torch.float16, device=device) for w in (d, 32)]
    kernel("paged_cache_read_f16")(key_elements, key_exponents, *values, i32([0, 64], device), *tables_[1:], *outs)
    assert torch.equal(outs[0][63].cpu(), plain64.dequantise(held[0], powers[0]).half()) and not outs[0][:63].any()


def test_captured(device):
    """An append captured in a graph writes what the buffers hold at each replay."""
    announce("cache append captured")
    keys, values = (cache(8, 4, 2, 64, True, device) for _ in range(2))
    k = torch.zeros((2, 2, 64), dtype=torch.float16, device=device)
    lengths = i32([1, 3], device)
    call = kernel("paged_cache_append_f16").prepare(k, k, *keys, *values, i32([0, 1, 2], device), i32([0, 2, 4], device),
                                                    i32([5, 0, 3, 7], device), lengths)
    graph = torch.cuda.CUDAGraph()
    call.launch()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call.launch()
    g = torch.Generator().manual_seed(5)
    for step in range(3):
        x = torch.randn((2, 2, 64), generator=g).half()
        k.copy_(x)
        before = (keys[0].clone(), keys[1].clone())
        graph.replay()
        torch.cuda.synchronize()
        at = [n - 1 for n in lengths.tolist()]
        slots = [([5, 0][at[0] // 4], at[0] % 4), ([3, 7][at[1] // 4], at[1] % 4)]
        want, powers = expected(before, x, slots)
        assert torch.equal(keys[0].contiguous().float().double().cpu(), want)
        assert torch.equal(keys[1].contiguous().int().cpu(), powers)
        lengths += 1


def test_append_as_a_torch_operator(device):
    """The cache is written in place through the operator's schema; a cache that shares storage with the rows is refused."""
    announce("cache append as a torch operator")
    g = torch.Generator().manual_seed(21)
    append = kernel("paged_cache_append_f16")
    held = [(*cache(3, 16, 2, 64, True, device), *cache(3, 16, 2, 64, True, device)) for _ in range(2)]
    k, v = (torch.randn((5, 2, 64), generator=g).half().to(device) for _ in range(2))
    tables_on = (i32([0, 2, 5], device), i32([0, 1, 2], device), i32([2, 0], device), i32([9, 3], device))
    append.run(k, v, *held[0], *tables_on)
    operation = append.as_torch_op("intent_amd_tests::paged_cache_append")
    assert operation(k, v, *held[1], *tables_on) is None
    for a, b in zip(*held):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    storage = torch.zeros(3 * 2 * 16 * 64 + 5 * 2 * 64 * 2, dtype=torch.uint8, device=device)
    shared = storage[:3 * 2 * 16 * 64].view(torch.float8_e4m3fn).view(3, 2, 16, 64).transpose(1, 2)
    rows = storage[3 * 2 * 16 * 64:].view(torch.float16).view(5, 2, 64)
    with pytest.raises(NotImplementedError):
        operation(rows, v, shared, *held[1][1:], *tables_on)
