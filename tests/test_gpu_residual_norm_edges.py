"""residual_norm, residual_norm_i8 and residual_norm_backward at rows and layouts that their other tests leave out."""
import pytest
import torch

from tests.gpu_util import announce
from tests.test_gpu_residual_norm import NUMBERS, case, kernel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("d", [72, 257, 4096])
def test_root_that_leaves_f32(device, d, post):
    """Rows whose mean square is infinite in f32 have a norm of 0, and rows whose mean square is 0 without an epsilon one of infinities: the
    8-bit rows say the same as the plain ones, 0 with a scale of 0, and a scale of NaN with elements of 0."""
    announce("residual_norm roots", d, post)
    given = [t.to(device) for t in case(d, "bf16", 6, d, False, post)]
    numbers = NUMBERS if post else (*NUMBERS[:2], 0.0)
    block, residual = given[0].clone(), given[1].clone()
    residual[1] *= 1e25
    block[2] *= 1e-30
    residual[2] = 1e-30
    run, run8 = kernel("residual_norm_bf16"), kernel("residual_norm_i8_bf16")
    total, out = run.run(block, residual, *given[2:5], *numbers)
    total8, elements, scales = run8.run(block, residual, *given[2:5], *numbers)
    assert torch.equal(total8, total)
    assert (out[1] == 0).all() and (elements[1] == 0).all() and scales[1] == 0
    for row in range(6):
        if out[row].isfinite().all() and (out[row] != 0).any():
            assert elements[row].abs().max() == 127 and scales[row] > 0 and scales[row].isfinite()
        elif not out[row].isfinite().all():
            assert (elements[row] == 0).all() and scales[row].isnan()
    if not post:
        assert out[2].isinf().all() and scales[2].isnan()
