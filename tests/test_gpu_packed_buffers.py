"""Written views that are slices of one packed buffer, element between element, give what separate buffers give and leave the rest
of the buffer alone; slices that share elements are refused, on the first call of a layout and on later ones."""
import pytest
import torch

from tests import test_gpu_linear_mxfp4 as linear
from tests import test_gpu_mx_cache as mx_cache
from tests import test_gpu_norm_rope as norm
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu


def test_keys_and_values_of_a_page_side_by_side(device):
    announce("packed cache")
    g = torch.Generator().manual_seed(1)
    i32 = mx_cache.i32
    pages, offsets, indices = mx_cache.tables([40, 7, 100], 16, g)
    tail = (i32([0, 40, 47, 147], device), i32(offsets, device), indices.to(device), i32([40, 7, 100], device))
    k, v = (torch.randn((147, 2, 64), generator=g).half().to(device) for _ in range(2))
    apart = [t for _ in range(2) for t in mx_cache.cache(pages, 16, 2, 64, False, device)]
    mx_cache.kernel("paged_cache_append_f16").run(k, v, *apart, *tail)
    elements = torch.full((pages, 3, 16, 2, 64), 0x55, dtype=torch.uint8, device=device)
    exponents = torch.full((pages, 3, 16, 2, 2), 121, dtype=torch.uint8, device=device)
    packed = [elements.view(torch.float8_e4m3fn)[:, 0], exponents[:, 0], elements.view(torch.float8_e4m3fn)[:, 1], exponents[:, 1]]
    append = mx_cache.kernel("paged_cache_append_f16")
    for _ in range(2):
        append.run(k, v, *packed, *tail)
        for got, want in zip(packed, apart):
            assert torch.equal(mx_cache.bits(got), mx_cache.bits(want))
        assert (elements[:, 2] == 0x55).all() and (exponents[:, 2] == 121).all()
        with pytest.raises(ValueError, match="overlap"):
            append.run(k, v, *packed[:2], *packed[:2], *tail)
    rows = torch.full((150, 5, 64), 3.0, dtype=torch.float16, device=device)
    mx_cache.kernel("paged_cache_read_f16")(*packed, *tail[:3], rows[:, :2], rows[:, 3:])
    outs = [torch.empty((150, 2, 64), dtype=torch.float16, device=device) for _ in range(2)]
    mx_cache.kernel("paged_cache_read_f16")(*apart, *tail[:3], *outs)
    assert torch.equal(rows[:147, :2], outs[0][:147]) and torch.equal(rows[:147, 3:], outs[1][:147])
    assert (rows[147:] == 3).all() and (rows[:, 2] == 3).all()


@pytest.mark.parametrize("d,pairs", [(128, 64), (96, 12)])
def test_gradients_of_a_packed_projection(device, d, pairs):
    announce("packed projection", d, pairs)
    rows, weights, positions, cos, sin, grad_q, grad_k = (t.to(device) for t in norm.case(2, "bf16", 65, 8, 2, d, pairs))
    common = (rows[:, :8], rows[:, 8:10], *weights, positions, cos, sin)
    want = norm.kernel("qk_norm_rope_backward_bf16").run(*common, grad_q, grad_k, norm.EPS)
    run, kept = norm.kernel("qk_norm_rope_backward_bf16"), norm.kernel("qk_norm_rope_bf16")
    packed, sums = torch.full_like(rows, 5.0), [torch.empty(d, device=device) for _ in range(2)]
    for _ in range(2):
        run(*common, grad_q, grad_k, packed[:, :8], packed[:, 8:10], *sums, norm.EPS)
        for got, exact in zip((packed[:, :8], packed[:, 8:10], *sums), want):
            assert torch.equal(got, exact)
        assert (packed[:, 10:] == 5).all()
        with pytest.raises(ValueError, match="overlap"):
            run(*common, grad_q, grad_k, packed[:, :8], packed[:, 7:9], *sums, norm.EPS)
    # rows turned within the projection's own buffer, behind what they are read from
    whole = torch.full((65, 24, d), 5.0, dtype=torch.bfloat16, device=device)
    whole[:, :10] = rows[:, :10]
    kept(whole[:, :8], whole[:, 8:10], *common[2:], whole[:, 10:18], whole[:, 18:20], norm.EPS)
    for got, exact in zip((whole[:, 10:18], whole[:, 18:20]), norm.kernel("qk_norm_rope_bf16").run(*common, norm.EPS)):
        assert torch.equal(got, exact)
    assert torch.equal(whole[:, :10], rows[:, :10]) and (whole[:, 20:] == 5).all()


def test_products_beside_their_rows(device):
    announce("packed rows and products")
    x, weight, exponents = (t.to(device) for t in linear.case(3, "f16", 33, 40, 96))
    want = linear.kernel("f16").run(x, weight, exponents)
    packed = torch.full((33, 160), 5.0, dtype=torch.float16, device=device)
    packed[:, :96] = x
    linear.kernel("f16")(packed[:, :96], weight, exponents, packed[:, 96:136])
    assert torch.equal(packed[:, 96:136], want) and torch.equal(packed[:, :96], x) and (packed[:, 136:] == 5).all()
    with pytest.raises(ValueError, match="overlap"):
        linear.kernel("f16")(packed[:, :96], weight, exponents, packed[:, 95:135])
