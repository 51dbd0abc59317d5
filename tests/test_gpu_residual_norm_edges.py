"""residual_norm, residual_norm_i8 and residual_norm_backward at rows and layouts that their other tests leave out."""
import pytest
import torch

from tests.gpu_util import announce
from tests.test_gpu_residual_norm import NUMBERS, case, close, kernel, plain

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


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 1021])
def test_special_rows_with_gates_and_a_block_norm(device, dtype, d):
    """Zeros, infinities and NaN in rows and gates stay in their rows; a sum that leaves f16 is an infinity, its norm formed before that."""
    announce("residual_norm special rows, gated", dtype, d)
    given = [t.to(device) for t in case(d, dtype, 12, d, True, True)]
    run, run8, back = (kernel(n + dtype) for n in ("residual_norm_", "residual_norm_i8_", "residual_norm_backward_"))
    want, want8 = run.run(*given[:5], *NUMBERS), run8.run(*given[:5], *NUMBERS)
    grads = back.run(given[0], want[0], *given[2:], *NUMBERS)
    block, residual, gate = (t.clone() for t in given[:3])
    block[0] = 0                                                       # a block of zeros under its norm adds nothing
    block[1, 5], residual[2, 7] = float("nan"), float("inf")
    gate[3], gate[4], gate[5] = float("nan"), float("inf"), 0
    block[6, 3] = float("inf")                                         # infinity over an infinite root
    residual[7] = 60000
    gate[7] = 40000
    moved = (block, residual, gate, *given[3:5])
    total, out = run.run(*moved, *NUMBERS)
    total8, elements, scales = run8.run(*moved, *NUMBERS)
    assert torch.equal(total8.isnan(), total.isnan()) and torch.equal(total8.nan_to_num(), total.nan_to_num())
    for got, other in ((total, want[0]), (out, want[1]), (elements, want8[1]), (scales, want8[2])):
        assert torch.equal(got[8:], other[8:])
    finite = [0, 5, 7]
    cpu = [t.cpu() for t in moved]
    h, h_size, y, y_size = plain(*(t[finite] for t in cpu[:3]), *cpu[3:])
    close(out[finite], y, y_size, dtype)
    inside = h.abs() < 60000
    close(total[finite].cpu()[inside], h[inside], h_size[inside], dtype)
    if dtype == "f16":
        assert (h[2].abs() > 70000).any() and total[7].cpu()[h[2].abs() > 70000].isinf().all()
    for row in (1, 3, 4, 6):
        assert not out[row].isfinite().all() and scales[row].isnan() and (elements[row] == 0).all()
    assert scales[2].isnan() and (elements[2] == 0).all()
    got = back.run(block, total, gate, *given[3:], *NUMBERS)
    for i in range(3):
        assert torch.equal(got[i][8:], grads[i][8:])
    for i in (3, 4):
        assert got[i].isnan().any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("at", range(5))
def test_gradients_along_themselves(device, dtype, at):
    """Along the signs of a gradient the change of the loss is the sum of its magnitudes, which half of the gradient, or one element in four
    left out, would miss by far more than the bound. A central difference of the 64-bit forward at 1e-4, off by 1e-8 / 6 of a third derivative.
    The kernel's gradient is off by a rounding of every element, and by what the rounding of the stored sum, from which it is formed, changes:
    half a step of magnitudes each, and as much again for the way through the norms."""
    announce("residual_norm gradients along themselves", dtype, at)
    half = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    given = case(5, dtype, 40, 64, True, True)
    on = [t.to(device) for t in given]
    total, _ = kernel("residual_norm_" + dtype).run(*on[:5], *NUMBERS)
    got = kernel("residual_norm_backward_" + dtype).run(on[0], total, *on[2:], *NUMBERS)[at].double().cpu()
    inputs = [t.double() for t in given[:5]]

    def value(s):
        moved = list(inputs)
        moved[at] = moved[at] + s * got.sign()
        h, _, y, _ = plain(*moved)
        return (h * given[5].double()).sum() + (y * given[6].double()).sum()

    slope = (value(1e-4) - value(-1e-4)) / 2e-4
    bound = 3 * half * got.abs().sum() + 1e-5 * got.numel()
    assert abs(got.abs().sum() - slope) <= bound
    assert abs(0.5 * got.abs().sum() - slope) > bound
    fewer = got.abs().flatten().clone()
    fewer[::4] = 0
    assert abs(fewer.sum() - slope) > bound


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 2304, 8200])
def test_nothing_is_written_beside_aligned_rows(device, dtype, d):
    """Outputs inside wider buffers whose rows begin at 16 bytes, which take whole pieces: the values of contiguous ones, and what lies beside
    them as it was."""
    announce("residual_norm beside aligned rows", dtype, d)
    given = [t.to(device) for t in case(3, dtype, 19, d, True, True)]
    total, _ = kernel("residual_norm_" + dtype).run(*given[:5], *NUMBERS)
    for name, inputs in (("residual_norm_", given[:5]), ("residual_norm_i8_", given[:5]),
                         ("residual_norm_backward_", (given[0], total, *given[2:]))):
        want = kernel(name + dtype).run(*inputs, *NUMBERS)
        whole = [torch.full((*t.shape[:-1], t.shape[-1] + 32), 7, dtype=t.dtype, device=device) for t in want]
        outs = [w[..., 16:16 + t.shape[-1]] for w, t in zip(whole, want)]
        kernel(name + dtype)(*inputs, *outs, *NUMBERS)
        for got, base, value in zip(outs, whole, want):
            assert torch.equal(got, value)
            assert (base[..., :16] == 7).all() and (base[..., -16:] == 7).all()
