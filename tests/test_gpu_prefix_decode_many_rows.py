"""paged_gqa_decode_prefix with so many query rows for a key head (more than four times their dimensions) that a wave takes two tiles of them."""
import pytest
import torch

from tests import prefix_weights
from tests.gpu_util import announce
from tests.test_gpu_prefix_decode import case, check, i32, kernel, run

pytestmark = pytest.mark.gpu

CASES = [
    # prefix, own lengths, query heads, key heads, d, page
    (300, [9] * 33, 16, 2, 64, 8), (200, [5, 0] * 37, 7, 1, 128, 20), (270, [33] * 40, 8, 1, 64, 32), (600, [50, 1] * 35, 32, 4, 128, 16),
    (31, [1] * 65, 16, 2, 128, 64), (1, [0, 2] * 44, 3, 1, 64, 16), (1021, [40, 300, 0] * 14, 13, 1, 128, 7), (64, [32, 64] * 17, 16, 2, 64, 16)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("size", [0.0, 1.0, 20.0])
@pytest.mark.parametrize("prefix,lengths,heads,kv_heads,d,ps", CASES)
def test_matches_plain_form(device, dtype, size, prefix, lengths, heads, kv_heads, d, ps):
    announce("decode behind a prefix, many rows", dtype, size, prefix, len(lengths), heads, kv_heads, d, ps)
    check(device, dtype, case(prefix, dtype, prefix, lengths, heads, kv_heads, d, ps, size=size))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("prefix,lengths,heads,kv_heads,d,ps", CASES)
def test_infinite_last_value(device, dtype, prefix, lengths, heads, kv_heads, d, ps):
    """Of the prefix's last token: in every sequence, and nothing else changes."""
    announce("decode behind a prefix, many rows, infinite last value", dtype, prefix, len(lengths), d, ps)
    given = case(prefix + d, dtype, prefix, lengths, heads, kv_heads, d, ps, size=0.5)
    want = run(device, dtype, given)
    group = heads // kv_heads
    for sign in (1.0, -1.0):
        values = given[2].clone()
        values[int(given[3][(prefix - 1) // ps]), (prefix - 1) % ps, 0, :3] = sign * float("inf")
        got = run(device, dtype, [*given[:2], values, *given[3:]])
        assert (got[:, :group, :3] == sign * float("inf")).all()
        keep = torch.ones(got.shape, dtype=torch.bool, device=device)
        keep[:, :group, :3] = False
        assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_all_scores_minus_infinity(device, dtype):
    announce("decode behind a prefix, many rows, all scores -inf", dtype)
    given = list(case(8, dtype, 45, [0, 3] * 17, 16, 2, 64, 16))
    given[0][:, :8] = given[0][:, :8].abs() + 0.5
    want = run(device, dtype, given)
    keys = given[1].clone()
    keys[:, :, 0] = float("-inf")
    got = run(device, dtype, [given[0], keys, *given[2:]])
    assert got[:, :8].isnan().all() and torch.equal(got[:, 8:], want[:, 8:])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("batch,group,d,ps", [(70, 4, 64, 16), (65, 8, 128, 32), (75, 7, 128, 7)])
def test_weights_take_part_whole(device, dtype, batch, group, d, ps):
    announce("decode behind a prefix, many rows, whole weights", dtype, batch, group, d, ps)
    heads = 8
    scores, values = prefix_weights.case(batch + d, dtype, heads, d)
    want, bound = prefix_weights.bar(scores, values, dtype)
    t = prefix_weights.TYPES[dtype]
    caches = [torch.zeros((2, ps, heads, d), dtype=t) for _ in range(2)]
    caches[0][1, :3, :, 5], caches[1][1, :3] = scores.to(t), values.to(t)
    q = torch.zeros((batch, heads * group, d), dtype=t)
    q[:, :, 5] = 1
    tables = [i32(x) for x in ([1], [3], [0] * (batch + 1), [], [0] * batch)]
    got = kernel(dtype, group).run(*(x.to(device) for x in (q, *caches, *tables)), 1.0).double().cpu()
    off = (got.unflatten(1, (heads, group)) - want[None, :, None]).abs() / bound[None, :, None]
    assert off.max() <= 1, off.max()
