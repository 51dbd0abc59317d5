"""linear_mxfp4 with weights past the type of x, which are infinite in it: sum_k x[m, k] W[n, k] by the rules of infinities, exactly
(x is a row of the unit matrix, so a result is one weight, or NaN where an infinite weight meets a 0)."""
import pytest
import torch

from tests import plain64
from tests.gpu_util import announce
from tests.test_gpu_linear_mxfp4 import TYPES, kernel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 9, 40, 150])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_infinite_weights(device, dtype, m):
    """Row n has the infinite element 6 (of either sign) at column n alone, rows 32 and 33 at two columns, row 34 nowhere."""
    announce("linear mxfp4 infinite weights", dtype, m)
    codes = torch.full((35, 32), 1, dtype=torch.uint8)                 # 0.5
    for n in range(32):
        codes[n, n] = 7 + 8 * (n % 2)
    codes[32, [3, 4]] = 7
    codes[33, [0, 31]] = torch.tensor([7, 15], dtype=torch.uint8)
    weight = codes[:, 0::2] | codes[:, 1::2] << 4
    exponents = torch.full((35, 1), 127 + (14 if dtype == "f16" else 126), dtype=torch.uint8)
    w = plain64.unpack_e2m1(weight, exponents).to(TYPES[dtype])
    assert w.isinf().sum() == 36
    x = torch.eye(32).repeat(5, 1)[:m].to(TYPES[dtype])
    got = kernel(dtype).run(x.to(device), weight.to(device), exponents.to(device)).cpu()
    for i in range(m):
        for n in range(35):
            others = torch.arange(32) != i % 32
            if w[n][others].isinf().any():
                assert got[i, n].isnan(), (i, n)
            else:
                assert got[i, n] == w[n, i % 32], (i, n)


@pytest.mark.parametrize("m", [1, 40, 150])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_every_infinite_row(device, dtype, m):
    """Every element at every exponent, twice a row: a row with an infinite weight is NaN throughout."""
    announce("linear mxfp4 infinite rows", dtype, m)
    code = torch.arange(32, dtype=torch.uint8) % 16
    packed, exponents = (code[0::2] | code[1::2] << 4).repeat(255, 1), torch.arange(255, dtype=torch.uint8)[:, None]
    x = torch.eye(32).repeat(5, 1)[:m].to(TYPES[dtype])
    finite = plain64.unpack_e2m1(packed, exponents).to(TYPES[dtype]).isfinite().all(1)
    got = kernel(dtype).run(x.to(device), packed.to(device), exponents.to(device)).cpu()
    assert (~finite).any() and got[:, ~finite].isnan().all() and got[:, finite].isfinite().all()
