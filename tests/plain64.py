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
