"""The bound of prefix_weights holds for f32 weights and not for bf16 weights of two numbers, 16 bits (CPU)."""
import pytest
import torch

from tests import prefix_weights


def output(scores, values, rounded, dtype):
    """The output with f32 weights that `rounded` has changed, and their sum, all else in 64 bits."""
    exponent = (scores * prefix_weights.LOG2E).float()
    weights = rounded(torch.exp2(exponent - exponent.amax(0))).double()
    return ((weights[:, :, None] * values).sum(0) / weights.sum(0)[:, None]).to(prefix_weights.TYPES[dtype])


def two_numbers(w):
    """The first 8 bits cut off, 8 more rounded."""
    high = (w.view(torch.int32) & ~0xFFFF).view(torch.float32)
    return high + (w - high).bfloat16().float()


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_whole_weights_pass(seed, dtype):
    scores, values = prefix_weights.case(seed, dtype, 32, 64)
    want, bound = prefix_weights.bar(scores, values, dtype)
    assert ((output(scores, values, lambda w: w, dtype).double() - want).abs() <= bound).all()


@pytest.mark.parametrize("seed", range(4))
def test_two_numbers_do_not(seed):
    scores, values = prefix_weights.case(seed, "bf16", 32, 64)
    want, bound = prefix_weights.bar(scores, values, "bf16")
    off = (output(scores, values, two_numbers, "bf16").double() - want).abs() / bound
    assert off.max() > 2 and (off > 1).double().mean() > 0.1
