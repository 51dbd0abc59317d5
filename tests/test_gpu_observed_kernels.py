"""The observation of a call names the kernel that its layout runs."""
import pytest
import torch

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
