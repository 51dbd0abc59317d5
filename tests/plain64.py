"""Plain 64-bit forms of the operators without a reference counterpart, written from their definitions (CPU, torch float64)."""
import torch


def rotate(x, positions, cos, sin, interleaved, back=False):
    """Rows [T, H, D] turned by their token's angles (back: turned back); positions are clamped into the tables."""
    out, pairs = x.clone(), cos.shape[1]
    if not pairs:
        return out
    at = positions.long().clamp(0, cos.shape[0] - 1)
    c, s = cos.double()[at][:, None], sin.double()[at][:, None] * (-1 if back else 1)
    first = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
    second = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    return out


def norm_rope(x, weight, positions, cos, sin, eps, interleaved):
    """(result, sum of the magnitudes that each element is formed from)."""
    x = x.double()
    y = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * weight.double()
    size = rotate(y.abs(), positions, cos.abs(), -sin.abs(), interleaved)           # a |c| + b |s| for the first of a pair
    other = rotate(y.abs(), positions, cos.abs(), sin.abs(), interleaved)
    return rotate(y, positions, cos, sin, interleaved), torch.maximum(size, other)


def norm_rope_backward(x, weight, grad, positions, cos, sin, eps, interleaved):
    """(grad_x, its magnitudes, grad_w, its magnitudes)."""
    x, weight, grad = x.double(), weight.double(), grad.double()
    g = rotate(grad, positions, cos, sin, interleaved, back=True)
    size = torch.maximum(rotate(grad.abs(), positions, cos.abs(), -sin.abs(), interleaved),
                         rotate(grad.abs(), positions, cos.abs(), sin.abs(), interleaved))
    r = 1 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    u = x * r
    inner, inner_size = g * weight, size * weight.abs()
    grad_x = r * (inner - u * (inner * u).mean(-1, keepdim=True))
    grad_size = r * (inner_size + u.abs() * (inner_size * u.abs()).mean(-1, keepdim=True))
    return grad_x, grad_size, (g * u).sum((0, 1)), (size * u.abs()).sum((0, 1))


def quantise(x):
    """Elements and exponent bytes of rows [..., D] in blocks of 32: the smallest e >= -127 with max |x| <= 448 * 2^e over
    the finite values, x * 2^-e rounded to e4m3 (four significant bits, multiples of 2^-9 below 2^-6, halves to even)."""
    blocks = x.double().unflatten(-1, (-1, 32))
    size = torch.where(blocks.isfinite(), blocks.abs(), 0.0).amax(-1)
    mantissa, exponent = torch.frexp(size)                       # size = mantissa * 2^exponent, mantissa in [0.5, 1)
    power = torch.where(size > 0, exponent - 9 + (mantissa > 0.875).int(), -127).clamp_min(-127)
    scaled = torch.ldexp(blocks, -power[..., None])
    _, at = torch.frexp(scaled)
    step = torch.ldexp(torch.ones_like(scaled), (at - 1).clamp_min(-6) - 3)
    elements = torch.where(blocks.isfinite(), torch.round(scaled / step) * step, float("nan"))
    return elements.flatten(-2), power + 127


def dequantise(elements, exponents):
    """What e4m3 elements (any float type) and exponent bytes stand for."""
    power = exponents.int() - 127
    scale = torch.where(exponents == 255, float("nan"), torch.ldexp(torch.ones(power.shape, dtype=torch.float64), power))
    return elements.double() * scale.repeat_interleave(32, -1)


def decode(q, keys, values, page_offsets, page_indices, lengths, scale):
    """q [B, HQ, D] over caches [P, PS, HK, D] of values (float64): (output, sum of weight * |value| over weights)."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    size = torch.zeros(q.shape, dtype=torch.float64)
    pages, ps, heads = keys.shape[:3]
    group = q.shape[1] // heads
    for b in range(q.shape[0]):
        slots = [(int(page_indices[i]), p) for i in range(int(page_offsets[b]), int(page_offsets[b + 1])) for p in range(ps)]
        slots = [(page, p) for page, p in slots[:max(0, int(lengths[b]))] if 0 <= page < pages]
        if not slots:
            continue
        at = torch.tensor(slots).unbind(1)
        for h in range(q.shape[1]):
            k, v = keys[at][:, h // group], values[at][:, h // group]
            weights = torch.softmax(k @ q[b, h].double() * scale, 0)
            out[b, h], size[b, h] = weights @ v, weights @ v.abs()
    return out, size


def unpack_e2m1(weight, exponents):
    """[N, K / 2] bytes and [N, K / 32] exponent bytes as float64 [N, K]."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    code = torch.stack((weight & 15, weight >> 4), -1).flatten(-2).long()
    return dequantise(torch.where(code >= 8, -table[code % 8], table[code % 8]), exponents)
