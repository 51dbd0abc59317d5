"""How far one-token attention that sums in f32 may be off, from each key's own error (CPU, torch float64).

Key j's score in the exponent of two is s_j = scale * log2(e) * (q . k_j), with a_j = |scale| * log2(e) * sum_d |q_d k_jd| >= |s_j|:
D exact products added in f32 (D + 2 roundings), log2(e), its product with the scale and the products with the sum (4), and the
difference from the running maximum, whose own score has rounded once more: (D + 8) * 2^-24 * a_j + 4 * 2^-24 * max a. exp2 is off
by 2^-22 with the factors that bring states together. So a weight is off by a share e_j, and sum p_j v_j by sum p_j e_j |v_j - out|.
The second product of 32 keys rounds 32 sums for each of up to three parts of a weight, once for a step of each of four waves, by
2^-23 each (sums that are cut off); 16 more join the states. Then half a step of the output type."""
import torch

HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f16": 2.0 ** -25, "bf16": 0.0}          # half the smallest subnormal
LOG2E = 1.4426950408889634


def tokens(keys, values, page_offsets, page_indices, length, b):
    """The keys and values [n, HK, D] of sequence b, in order."""
    pages, ps = keys.shape[:2]
    slots = [(int(page_indices[i]), p) for i in range(int(page_offsets[b]), int(page_offsets[b + 1])) for p in range(ps)]
    slots = [(page, p) for page, p in slots[:max(0, int(length))] if 0 <= page < pages]
    if not slots:
        return keys.reshape(-1, *keys.shape[2:])[:0], values.reshape(-1, *values.shape[2:])[:0]
    at = torch.tensor(slots).unbind(1)
    return keys[at], values[at]


def bar(q, keys, values, page_offsets, page_indices, lengths, scale, dtype):
    """(output, bound on what a kernel's may be off), both [B, HQ, D]."""
    q = q.double()
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    d, group = q.shape[2], q.shape[1] // keys.shape[2]
    for b in range(q.shape[0]):
        k, v = tokens(keys, values, page_offsets, page_indices, lengths[b], b)
        if not len(k):
            continue
        rounds = 3 * 32 * -(-len(k) // 128) + 16
        for h in range(q.shape[1]):
            kh, vh = k[:, h // group], v[:, h // group]
            p = torch.softmax(kh @ q[b, h] * scale, 0)
            a = abs(scale) * LOG2E * (kh.abs() @ q[b, h].abs())
            error = 0.6932 * ((d + 8) * 2.0 ** -24 * a + 4 * 2.0 ** -24 * a.max()) + 2.0 ** -22
            out[b, h] = p @ vh
            bound[b, h] = (p * error) @ (vh - out[b, h]).abs() + rounds * 2.0 ** -23 * (p @ vh.abs())
    return out, bound * 1.001 + HALF_STEP[dtype] * out.abs() + LEAST[dtype]


def check(got, want, bound):
    got = got.double().cpu()
    assert not got.isnan().any()
    over = (got - want).abs() - bound
    assert (over <= 0).all(), f"off by {(got - want).abs().flatten()[over.argmax()]} of {want.flatten()[over.argmax()]}"


def sink(g, count, d, heads, group, bits, size):
    """Queries, keys and values (float64) of one sequence whose first key outweighs each of the others by 2^bits and has the
    value 0, and the scale that does it. Values are `size` to twice that, of four bits, so the output is the others' share."""
    direction = torch.randint(0, 2, (d,), generator=g).double() * 2 - 1
    keys = torch.randint(-1, 2, (count, heads, d), generator=g).double() / 64
    keys[0] = direction
    values = size * (1 + torch.randint(0, 8, (count, heads, d), generator=g).double() / 8)
    values[0] = 0
    return direction.expand(1, heads * group, d).clone(), keys, values, float(torch.tensor(bits / (d * LOG2E), dtype=torch.float32))
