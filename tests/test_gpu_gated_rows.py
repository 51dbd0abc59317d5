"""swiglu_quantize_rows at the ends of bf16: gates whose e^-g or product with log2(e) leaves f32, infinities and NaN."""
import pytest
import torch

from tests.gpu_util import announce
from tests.test_gpu_linear_i8 import kernel

pytestmark = pytest.mark.gpu


def test_ends_of_the_type(device):
    announce("gated rows, ends of the type")
    gate = torch.tensor([[3e38, -3e38, 1.0, -1e30], [-1e4, -200.0, -3e38, 2.0], [float("inf"), 1.0, 1.0, 1.0], [float("-inf"), 1.0, 1.0, 1.0],
                         [float("nan"), 1.0, 1.0, 1.0], [-1e4, -200.0, -3e38, -1e30]]).bfloat16()
    up = torch.full_like(gate, 0.5)
    elements, scales = kernel("swiglu_quantize_rows_bf16").run(gate.to(device), up.to(device))
    want = torch.tensor([[127, 0, 0, 0], [0, 0, 0, 127]] + [[0] * 4] * 4, dtype=torch.int8)
    assert torch.equal(elements.cpu(), want)
    assert scales[2:5].isnan().all() and scales[5] == 0 and scales[:2].isfinite().all() and (scales[:2] > 0).all()
