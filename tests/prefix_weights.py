"""Attention behind a shared prefix whose output shows how many bits of a weight took part (CPU, torch float64).

Three tokens a head, of weights near a third each, whose values cancel: the second value is what the first's share leaves, rounded to the
rows' type, and the third what both leave. The output is then about 2^-2b of the values (b bits of the type), its rounding far below f32's of
a weight, and an error of a weight stands out in it.

Bound. A score is one product, exact; the factor scale * log2(e) is off by two roundings and its product with the score by one more: 3 * 2^-24
of a_j = |score| * log2(e). The sum with the peak rounds once, by half a step of a number below 2 (bf16) or below 16 (f16, whose weights are held
near 2^12). exp2 is off by 2^-22. So a weight is off by a share e_j, and the output by sum p_j e_j |v_j - out|. Three tokens of three numbers each are
9 terms, each rounding by 2^-23 of the magnitudes (sums that are cut off); the divisor's sum and the division add 3. Then half a step of the type."""
import torch

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f16": 2.0 ** -25, "bf16": 1e-40}
PEAK_STEP = {"f16": 2.0 ** -21, "bf16": 2.0 ** -24}
LOG2E = 1.4426950408889634


def case(seed, dtype, heads, d):
    """Scores [3, heads], and values [3, heads, d] of the type, in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    scores = torch.randint(-128, 129, (3, heads), generator=g).double() / 256
    p = torch.softmax(scores, 0)
    first = (32 * (1 + torch.rand((heads, d), generator=g))).to(TYPES[dtype]).double()
    second = (-p[0][:, None] * first / p[1][:, None]).to(TYPES[dtype]).double()
    left = p[0][:, None] * first + p[1][:, None] * second
    third = (-left / p[2][:, None]).to(TYPES[dtype]).double()
    return scores, torch.stack((first, second, third))


def bar(scores, values, dtype):
    """(output, bound on what a kernel's may be off), both [heads, d]."""
    p = torch.softmax(scores, 0)
    error = 0.6932 * (3 * 2.0 ** -24 * scores.abs() * LOG2E + PEAK_STEP[dtype]) + 2.0 ** -22
    out = (p[:, :, None] * values).sum(0)
    bound = ((p * error)[:, :, None] * (values - out).abs()).sum(0) + 12 * 2.0 ** -23 * (p[:, :, None] * values.abs()).sum(0)
    return out, bound * 1.001 + HALF_STEP[dtype] * out.abs() + LEAST[dtype]
