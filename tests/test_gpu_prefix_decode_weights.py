"""paged_gqa_decode_prefix takes its weights whole: values that cancel, so that the output is what rounding leaves. The bound is that of
prefix_weights.py, which 16 bits of a weight do not keep."""
import pytest
import torch

from tests import prefix_bar, prefix_weights
from tests.gpu_util import announce
from tests.test_gpu_prefix_decode import case, i32, kernel, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("batch,group,d,ps,shared", [
    (1, 1, 64, 16, True), (2, 3, 128, 32, True), (40, 5, 64, 16, True), (40, 4, 128, 16, True), (30, 8, 128, 7, True),
    (1, 1, 128, 16, False), (3, 5, 64, 32, False), (9, 17, 128, 7, False)])
def test_weights_take_part_whole(device, dtype, batch, group, d, ps, shared):
    announce("decode behind a prefix, whole weights", dtype, batch, group, d, ps, shared)
    heads = 8
    scores, values = prefix_weights.case(batch + d, dtype, heads, d)
    want, bound = prefix_weights.bar(scores, values, dtype)
    t = prefix_weights.TYPES[dtype]
    caches = [torch.zeros((2, ps, heads, d), dtype=t) for _ in range(2)]
    caches[0][1, :3, :, 5], caches[1][1, :3] = scores.to(t), values.to(t)
    q = torch.zeros((batch, heads * group, d), dtype=t)
    q[:, :, 5] = 1
    tables = ([1], [3], [0] * (batch + 1), [], [0] * batch) if shared else ([], [0], range(batch + 1), [1] * batch, [3] * batch)
    got = kernel(dtype, group).run(*(x.to(device) for x in (q, *caches, *(i32(list(x)) for x in tables))), 1.0).double().cpu()
    off = (got.unflatten(1, (heads, group)) - want[None, :, None]).abs() / bound[None, :, None]
    assert off.max() <= 1, off.max()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("bits", [12, 20, 26, 30])
@pytest.mark.parametrize("prefix,own", [(200, 50), (1, 300), (300, 0)])
def test_outweighed_by_one(device, dtype, bits, prefix, own):
    """The first key outweighs the others by about 2^bits and has a value of 0, and the others' values are of one sign, so what a weight is off by
    adds up. A weight is off by its own share and in f16 by that type's last, 2^-24, where the largest is at least 2^11.9; else as prefix_bar has
    it."""
    announce("decode behind a prefix, outweighed, one sign", dtype, bits, prefix, own)
    given = list(case(4, dtype, prefix, [own], 4, 2, 64, 16))
    q, keys, values = given[:3]
    direction = torch.where(torch.arange(64) % 3 == 0, -1.0, 1.0)
    q[:] = direction
    keys[:] = (torch.randint(-1, 2, keys.shape, generator=torch.Generator().manual_seed(1)) / 64).to(keys.dtype)
    values[:] = values.abs() + 0.5
    first = int(given[3][0])
    keys[first, 0], values[first, 0] = direction.to(keys.dtype), 0
    given[8] = float(torch.tensor(bits / (64 * prefix_bar.LOG2E)))
    out, _ = prefix_bar.bar(*given, dtype)
    got = run(device, dtype, given).double().cpu()
    k, v = (torch.cat((prefix_bar.rows(c.double(), given[3], 0, len(given[3]), prefix),
                       prefix_bar.rows(c.double(), given[6], 0, len(given[6]), own))) for c in given[1:3])
    heads = torch.arange(4) // 2
    p = torch.softmax(torch.einsum("thd,hd->ht", k[:, heads], q[0].double()) * given[8], -1)
    a = given[8] * prefix_bar.LOG2E * torch.einsum("thd,hd->ht", k[:, heads].abs(), q[0].double().abs())
    error = 0.6932 * (72 * 2.0 ** -24 * a + 4 * 2.0 ** -24 * a.amax(-1, keepdim=True) + prefix_weights.PEAK_STEP[dtype]) + 2.0 ** -22
    share = p * error + (2.0 ** -35.9 if dtype == "f16" else 0)
    weighted = torch.einsum("ht,thd->hd", share, (v[:, heads] - out[0]).abs())
    rounds = (3 * 32 * -(-len(k) // 32) + 80) * 2.0 ** -23 * torch.einsum("ht,thd->hd", p, v[:, heads].abs())
    bound = 1.001 * (weighted + rounds) + prefix_bar.HALF_STEP[dtype] * out[0].abs() + prefix_bar.LEAST[dtype]
    off = (got[0] - out[0]).abs() / bound
    assert off.max() <= 1, off.max()
