"""qk_norm_rope and its backward at the ends of their ranges: no eps, and the bars of tests/test_gpu_norm_rope.py."""
import pytest
import torch

from tests import plain64
from tests.gpu_util import announce
from tests.test_gpu_norm_rope import case, close, kernel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,q_heads,kv_heads,d,pairs,interleaved", [
    (33, 5, 1, 64, 16, False), (7, 32, 8, 64, 32, True), (3, 3, 0, 128, 64, False), (300, 7, 2, 96, 24, False),
    (5, 1, 1, 256, 128, True), (9, 2, 1, 20, 3, False)])
def test_without_eps(device, dtype, tokens, q_heads, kv_heads, d, pairs, interleaved):
    """Rows that are not zero need no eps; numbers of heads that leave a part of a wave without a row, in both row kernels."""
    announce("qk_norm_rope without eps", dtype, tokens, q_heads, kv_heads, d)
    rows, weights, positions, cos, sin, grad_q, grad_k = case(tokens + d, dtype, tokens, q_heads, kv_heads, d, pairs)
    heads = slice(0, q_heads), slice(q_heads, q_heads + kv_heads)
    on = rows.to(device)
    common = (on[:, heads[0]], on[:, heads[1]], *weights.to(device), positions.to(device), cos.to(device), sin.to(device))
    out = kernel(f"qk_norm_rope_{dtype}", interleaved).run(*common, 0.0)
    got = kernel(f"qk_norm_rope_backward_{dtype}", interleaved).run(*common, grad_q.to(device), grad_k.to(device), 0.0)
    for i, grad in enumerate((grad_q, grad_k)):
        x = rows[:, heads[i]]
        if x.numel():
            want, size = plain64.norm_rope(x, weights[i], positions, cos, sin, 0.0, interleaved)
            close(out[i], want, size, dtype, 2.0 ** -18)
            dx, dx_size, dw, dw_size = plain64.norm_rope_backward(x, weights[i], grad, positions, cos, sin, 0.0, interleaved)
            close(got[i], dx, dx_size, dtype, 2.0 ** -17)
            assert ((got[2 + i].double().cpu() - dw).abs() <= 2.0 ** -15 * dw_size + 1e-37).all()
        else:
            assert (got[2 + i] == 0).all()


@pytest.mark.parametrize("absent", [0, 1])
def test_absent_heads_of_any_layout(device, absent):
    """The heads that are not there have no layout to refuse."""
    announce("qk_norm_rope absent heads", absent)
    rows, weights, positions, cos, sin, grad, _ = (t.to(device) for t in case(7, "bf16", 5, 3, 1, 64, 32))
    x, nothing = rows[:, :3], torch.empty((5, 0, 64, 2), dtype=torch.bfloat16, device=device)[..., 0]
    both = lambda a: (nothing, a) if absent == 0 else (a, nothing)          # noqa: E731
    common = (*both(x), *weights, positions, cos, sin)
    plain = (*both(x.contiguous()), *weights, positions, cos, sin)
    out = kernel("qk_norm_rope_bf16").run(*common, 1e-6)
    none = torch.empty((5, 0, 64), dtype=torch.bfloat16, device=device)
    want = kernel("qk_norm_rope_bf16").run(*[none if t is nothing else t for t in plain], 1e-6)
    assert torch.equal(out[1 - absent], want[1 - absent]) and out[absent].shape == (5, 0, 64)
    got = kernel("qk_norm_rope_backward_bf16").run(*common, *both(grad), 1e-6)
    sizes = [t.abs().sum().item() for t in got[2:]]
    assert sizes[absent] == 0 and sizes[1 - absent] > 0 and got[1 - absent].isfinite().all()
