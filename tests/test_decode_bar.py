"""That the bar of one-token attention tells a kernel with whole weights from ones that leave bits of them out: the second product is
formed here, on the CPU, from what a kernel would take of each weight."""
import pytest
import torch

from tests import decode_bar

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def cut(w, bits, least):
    """w cut off, toward 0, to `bits` bits and multiples of `least`."""
    _, at = torch.frexp(w)
    step = torch.maximum(torch.ldexp(torch.ones_like(w), at - bits), torch.full_like(w, least))
    return torch.floor(w / step) * step


WHOLE = lambda w: w.float().double()                                                        # noqa: E731
ONE_BF16 = lambda w: w.bfloat16().double()                                                  # noqa: E731
ONE_F16 = lambda w: cut(w, 11, 2.0 ** -24)                                                  # noqa: E731
TWO_F16 = lambda w: cut(w, 11, 2.0 ** -24) + cut(w - cut(w, 11, 2.0 ** -24), 11, 2.0 ** -24)    # noqa: E731


def formed(q, keys, values, scale, dtype, taken):
    """One sequence's output with the weights that `taken` leaves of those against the largest; the divisor has them whole."""
    group, out = q.shape[1] // keys.shape[1], torch.zeros(q.shape, dtype=torch.float64)
    for h in range(q.shape[1]):
        s = keys[:, h // group] @ q[0, h].double() * scale
        w = torch.exp(s - s.max())
        out[0, h] = taken(w) @ values[:, h // group] / WHOLE(w).sum()
    return out.to(TYPES[dtype])


def caught(got, want, bound):
    return bool(((got.double() - want).abs() > bound).any())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,heads,group,d", [(40, 2, 4, 64), (100, 2, 2, 128), (128, 1, 5, 64)])
def test_weights_of_even_scores(dtype, n, heads, group, d):
    """Near-even weights: one bf16 number of each is caught, whole weights pass."""
    g = torch.Generator().manual_seed(n)
    keys = torch.randint(-8, 9, (n, heads, d), generator=g).double() / 64
    values = torch.randint(-15, 16, (n, heads, d), generator=g).double() / 8
    q = torch.randn((1, heads * group, d), generator=g).to(TYPES[dtype])
    scale = 2.0 ** -4
    at = (keys[None], values[None], [0, 1], [0], [n], scale, dtype)
    want, bound = decode_bar.bar(q, *at)
    assert not caught(formed(q, keys, values, scale, dtype, WHOLE), want, bound)
    assert caught(formed(q, keys, values, scale, dtype, ONE_BF16), want, bound)
    if dtype == "f16" and n < 100:
        assert caught(formed(q, keys, values, scale, dtype, ONE_F16), want, bound)


@pytest.mark.parametrize("bits,size", [(18, 2.0), (20.3, 2.0), (22.5, 32.0), (24.5, 128.0), (28, 1024.0)])
def test_weights_against_one_that_outweighs_them(bits, size):
    """What one key with the value 0 leaves to the others: two f16 numbers of a weight, which end at 2^-24, are caught."""
    g = torch.Generator().manual_seed(int(bits * 10))
    q, keys, values, scale = decode_bar.sink(g, 700, 64, 2, 2, bits, size)
    want, bound = decode_bar.bar(q, keys[None], values[None], [0, 1], [0], [700], scale, "f16")
    assert not caught(formed(q, keys, values, scale, "f16", WHOLE), want, bound)
    assert caught(formed(q, keys, values, scale, "f16", TWO_F16), want, bound)
