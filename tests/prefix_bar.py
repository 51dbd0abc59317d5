"""How far one-token attention behind a shared prefix may be off, from each key's own error (CPU, torch float64).

Key j's score in the exponent of two is s_j = scale * log2(e) * (q . k_j), with a_j = |scale| * log2(e) * sum_d |q_d k_jd| >= |s_j|: D exact
products added in f32 (D + 2 roundings), log2(e), its product with the scale and the products with the sum (4), and the difference from the
peak, whose own score has rounded once more: (D + 8) * 2^-24 * a_j + 4 * 2^-24 * max a. exp2 is off by 2^-22 with the factors that bring
states together. A weight is rounded by 2^-16 of itself (two bf16 numbers: 8 bits cut off, 8 more rounded) or 2^-21 (two f16 numbers) and
2^-36 of the largest; the sum that divides is of the same. So a weight is off by a share e_j, and sum p_j v_j by sum p_j e_j |v_j - out|.
The second product of 32 keys rounds 32 sums for each of two parts of a weight, by 2^-23 each (sums that are cut off), over all steps of a
wave's walk; 80 more join the states. Then half a step of the output type."""
import torch

HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f16": 2.0 ** -25, "bf16": 1e-40}
ROUNDED = {"f16": 2.0 ** -21, "bf16": 2.0 ** -16}
LOG2E = 1.4426950408889634


def rows(cache, pages, first, count, length):
    """The first `length` tokens [n, HK, D] of `count` entries of `pages` from `first` on, entries and pages clamped into their arrays."""
    ps = cache.shape[1]
    length = min(max(int(length), 0), max(int(count), 0) * ps)
    if not length or not cache.shape[0]:
        return cache.reshape(-1, *cache.shape[2:])[:0]
    at = (torch.arange(length) // ps + int(first)).clamp(0, len(pages) - 1)
    return cache[pages.long()[at].clamp(0, cache.shape[0] - 1), torch.arange(length) % ps]


def bar(q, keys, values, prefix_indices, prefix_length, page_offsets, page_indices, lengths, scale, dtype):
    """(output, bound on what a kernel's may be off), both [B, HQ, D]."""
    q, keys, values = q.double(), keys.double(), values.double()
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    d, group = q.shape[2], q.shape[1] // keys.shape[2]
    shared = [rows(c, prefix_indices, 0, len(prefix_indices), prefix_length) for c in (keys, values)]
    for b in range(q.shape[0]):
        first, count = page_offsets[b], page_offsets[b + 1] - page_offsets[b]
        k, v = (torch.cat((old, rows(c, page_indices, first, count, lengths[b]))) for old, c in zip(shared, (keys, values)))
        if not len(k):
            continue
        rounds = 2 * 32 * -(-len(k) // 32) + 80
        heads = torch.arange(q.shape[1]) // group
        kh, vh = k[:, heads].transpose(0, 1).contiguous(), v[:, heads].transpose(0, 1).contiguous()        # [HQ, T, D]
        p = torch.softmax((kh @ q[b][:, :, None])[..., 0] * scale, -1)
        a = abs(scale) * LOG2E * (kh.abs() @ q[b].abs()[:, :, None])[..., 0]
        error = 0.6932 * ((d + 8) * 2.0 ** -24 * a + 4 * 2.0 ** -24 * a.amax(-1, keepdim=True)) + 2.0 ** -22 + ROUNDED[dtype]
        out[b] = (p[:, None] @ vh)[:, 0]
        share = p * error + 2.0 ** -36 * p.amax(-1, keepdim=True)
        bound[b] = (share[:, None] @ (vh - out[b][:, None]).abs())[:, 0] + rounds * 2.0 ** -23 * (p[:, None] @ vh.abs())[:, 0]
    return out, bound * 1.001 + HALF_STEP[dtype] * out.abs() + LEAST[dtype]


def check(got, want, bound):
    got = got.double().cpu()
    assert not got.isnan().any()
    over = (got - want).abs() - bound
    assert (over <= 0).all(), f"off by {(got - want).abs().flatten()[over.argmax()]} of {want.flatten()[over.argmax()]}"
