"""paged_gqa_decode_prefix takes its weights whole: values that cancel, so that the output is what rounding leaves. The bound is that of
prefix_weights.py, which 16 bits of a weight do not keep."""
import pytest
import torch

from tests import prefix_weights
from tests.gpu_util import announce
from tests.test_gpu_prefix_decode import i32, kernel

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
