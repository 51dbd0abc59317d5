"""The observation of a call names the kernel that its layout runs."""
import pytest
import torch

from tests import test_gpu_norm_rope as norm
from tests.gpu_util import announce
from tests.test_gpu_mx_cache import cache, i32
from tests.test_gpu_mx_decode import kernel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stride,walk", [(64, "true"), (2 ** 26 - 16, "true"), (2 ** 26, "false")])
def test_decode_of_far_tokens(device, stride, walk):
    """Tokens so far apart that a lane's place in a tile passes 32 bits are walked one by one."""
    announce("observed decode", stride)
    store = torch.zeros(15 * stride + 2 * 64, dtype=torch.uint8, device=device)
    far = store.as_strided((2, 16, 1, 64), (64, stride, 64, 1)).view(torch.float8_e4m3fn)
    near, powers = cache(2, 16, 1, 64, False, device)
    q = torch.ones((1, 4, 64), dtype=torch.float16, device=device)
    tables = (i32([0, 2], device), i32([0, 1], device), i32([20], device))
    for held in ((far, powers, near, powers), (near, powers, far, powers)):
        call = kernel("f16", 4).prepare(q, *held, *tables, 1.0)
        call.launch()
        assert f",1,{walk}," in call.observation.kernel, call.observation.kernel


@pytest.mark.parametrize("absent", [0, 1])
def test_norm_of_absent_heads(device, absent):
    """The weight of heads that are not there says nothing about the kernel, however it lies."""
    announce("observed norm", absent)
    rows, weights, positions, cos, sin, grad, _ = (t.to(device) for t in norm.case(7, "bf16", 5, 3, 1, 64, 32))
    odd = torch.ones(65, device=device)[1:]
    both = lambda a, b: (b, a) if absent == 0 else (a, b)          # noqa: E731
    none = torch.empty((5, 0, 64), dtype=torch.bfloat16, device=device)
    common = (*both(rows[:, :3], none), *both(weights[0], odd), positions, cos, sin)
    for name, grads in (("qk_norm_rope_bf16", ()), ("qk_norm_rope_backward_bf16", both(grad, none))):
        call = norm.kernel(name).prepare(*common, *grads, 1e-6)
        call.launch()
        assert "_rows<" in call.observation.kernel, call.observation.kernel
