"""paged_gqa_decode_mx where the weights' own bits matter: near-even weights and weights far below the largest, held to what each
key's error allows (tests/decode_bar.py); and values at the ends of f16."""
import pytest
import torch

from tests import decode_bar, plain64
from tests.gpu_util import announce
from tests.test_gpu_mx_cache import cache, i32
from tests.test_gpu_mx_decode import TYPES, kernel

pytestmark = pytest.mark.gpu


def held(rows, page, device, exact=True):
    """A cache whose pages, in order, hold rows [n, HK, D] (float64; exact: without a rounding) and what it stands for."""
    pages = -(-rows.shape[0] // page)
    out = cache(pages, page, rows.shape[1], rows.shape[2], True, device, 0x7F)
    padded = torch.zeros((pages * page, *rows.shape[1:]), dtype=torch.float64)
    padded[:rows.shape[0]] = rows
    padded = padded.unflatten(0, (pages, page))
    elements, powers = plain64.quantise(padded)
    plain = plain64.dequantise(elements, powers)
    assert not exact or torch.equal(plain, padded)
    out[0].view(torch.uint8).copy_(elements.float().to(torch.float8_e4m3fn).view(torch.uint8))
    out[1].copy_(powers.to(torch.uint8))
    return out, plain


def run(q, keys, values, page, scale, dtype, device, exact=True):
    n, heads = keys.shape[:2]
    group = q.shape[1] // heads
    (key_cache, plain_keys), (value_cache, plain_values) = held(keys, page, device), held(values, page, device, exact)
    pages = plain_keys.shape[0]
    out = kernel(dtype, group).run(q.to(TYPES[dtype]).to(device), *key_cache, *value_cache, i32([0, pages], device),
                                   torch.arange(pages, dtype=torch.int32, device=device), i32([n], device), scale)
    return out, (plain_keys, plain_values, [0, pages], list(range(pages)), [n], scale, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,heads,group,d,page", [(40, 2, 4, 64, 16), (100, 2, 2, 128, 64), (128, 1, 5, 64, 16), (100, 1, 20, 96, 16),
                                                  (70, 2, 3, 192, 8), (61, 1, 3, 256, 16), (100, 1, 33, 64, 5)])
def test_even_scores(device, dtype, n, heads, group, d, page):
    announce("mx decode even scores", dtype, n, heads, group, d, page)
    g = torch.Generator().manual_seed(n + page)
    keys = torch.randint(-8, 9, (n, heads, d), generator=g).double() / 64
    values = torch.randint(-15, 16, (n, heads, d), generator=g).double() / 8
    q = torch.randn((1, heads * group, d), generator=g).to(TYPES[dtype])
    out, at = run(q, keys, values, page, 2.0 ** -4, dtype, device)
    decode_bar.check(out, *decode_bar.bar(q, *at))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("bits,size", [(18, 2.0), (20.3, 2.0), (22.5, 32.0), (24.5, 128.0), (28, 1024.0), (34, 8192.0)])
@pytest.mark.parametrize("n,d,page", [(700, 64, 16), (3000, 128, 64), (700, 64, 5)])
def test_one_key_outweighs_the_others(device, dtype, bits, size, n, d, page):
    """The first key outweighs the others by 2^bits and has the value 0: what is left is theirs, to its own precision. In one job
    and in many, with pages of any size; the larger values have exponents that f16's range makes the kernel look at."""
    announce("mx decode outweighed", dtype, bits, n, d, page)
    g = torch.Generator().manual_seed(int(bits * 10))
    q, keys, values, scale = decode_bar.sink(g, n, d, 2, 2, bits, size)
    out, at = run(q, keys, values, page, scale, dtype, device)
    decode_bar.check(out, *decode_bar.bar(q, *at))


@pytest.mark.parametrize("page", [16, 8])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_values_at_the_ends_of_f16(device, d, page):
    """Values are taken in the query's type: f16 rounds those below 2^-14 to multiples of 2^-24 and has none past 65504, in every
    block of a row by its own exponent; a bf16 query has them all."""
    announce("mx decode ends of f16", d, page)
    g = torch.Generator().manual_seed(d + page)
    keys = torch.zeros((40, 1, d), dtype=torch.float64)
    values = torch.randint(1, 16, (40, 1, d), generator=g).double() / 8
    values[..., :32] *= 2.0 ** 14                     # up to 1.875 * 2^14
    values[..., 32:64] *= 2.0 ** -25                  # multiples of 2^-28
    for dtype in ("f16", "bf16"):
        q = torch.ones((1, 2, d), dtype=TYPES[dtype])
        out, (plain_keys, plain_values, *at) = run(q, keys, values, page, 1.0, dtype, device)
        decode_bar.check(out, *decode_bar.bar(q, plain_keys, plain_values.to(TYPES[dtype]).double(), *at))
    values[7, 0, 3] = 2.0 ** 16
    f16, _ = run(torch.ones((1, 2, d)), keys, values, page, 1.0, "f16", device)
    bf16, _ = run(torch.ones((1, 2, d)), keys, values, page, 1.0, "bf16", device)
    assert f16[..., 3].isposinf().all() and f16.isfinite().sum() == f16.numel() - 2 and bf16.isfinite().all()
    values[:] = 1.25 * 2.0 ** -24                     # one step of f16, where the sum of 40 of them would round to it as well
    alone, _ = run(torch.ones((1, 2, d)), keys[:1], values[:1], page, 1.0, "f16", device)
    assert (alone.double() == 2.0 ** -24).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page", [16, 8])
def test_infinite_values(device, dtype, page):
    """A value past its type is an infinity of the heads and the column that see it, whatever bits the weights have."""
    announce("mx decode infinite values", dtype, page)
    keys = torch.zeros((40, 2, 64), dtype=torch.float64)
    keys[5, 0] = 1 / 8
    values = torch.ones((40, 2, 64), dtype=torch.float64)
    largest = 2.0 ** 16 if dtype == "f16" else 448 * 2.0 ** 120
    values[7, 1, 40], values[9, 0, 3] = largest, -largest
    q = torch.ones((1, 4, 64), dtype=torch.float64) * torch.tensor([0.0, 0.7, 0.0, 0.3])[:, None]
    out, _ = run(q, keys, values, page, 0.1, dtype, device, exact=False)       # beside 2^128, a block's ones are 0
    assert out[0, 2:, 40].isposinf().all() and out[0, :2, 3].isneginf().all()
    assert out.isfinite().sum() == out.numel() - 4


def test_long_table_without_a_page(device):
    """A table too long for one job over a cache that has no page: 0 from every job."""
    announce("mx decode long table, no page")
    held = [torch.zeros((0, 64, 8, w), dtype=torch.uint8, device=device) for w in (64, 2, 64, 2)]
    held[0], held[2] = held[0].view(torch.float8_e4m3fn), held[2].view(torch.float8_e4m3fn)
    q = torch.ones((4, 32, 64), dtype=torch.float16, device=device)
    out = torch.full_like(q, 7.0)
    kernel("f16", 4)(q, *held, i32([0, 10, 20000, 20000, 50001], device), torch.zeros(50001, dtype=torch.int32, device=device),
                     i32([640, 10 ** 6, 5, 2 * 10 ** 6], device), out, 1.0)
    assert (out == 0).all()
