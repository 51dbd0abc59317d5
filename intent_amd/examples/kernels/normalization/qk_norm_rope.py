"""Root-mean-square norm of every query and key head with the rotation of its token's position, in one pass over the
projected rows: `qk_norm_rope_f16` and `qk_norm_rope_bf16`. No reference counterpart.

For a head's row x of width D at a token of position p, weight w (of the queries or of the keys), R rotated pairs and
tables cos, sin:

  y_d      = x_d * rsqrt(mean(x^2) + eps) * w_d                     f32
  (a, b)   = (y_i, y_{i + R}), or with INTERLEAVED (y_2i, y_2i+1),  i < R
  (a', b') = (a cos[p, i] - b sin[p, i], b cos[p, i] + a sin[p, i])
  out      = the rotated pairs in their places, y_d for d >= 2R, stored in the storage type

2R <= D; R = 0 is the norm alone. A position outside the tables takes their nearest row.

The bodies state this one token at a time; the hip provider recognises a definition by name and signature.
"""
import intent_amd as intent
import intent_amd.language as I


@intent.fn
def rotation_partners(D, R, interleaved):
    """Per dimension: the other dimension of its pair (itself where none), the pair, and the sign of the partner's sine."""
    d = I.indices(I.domain(0, D))
    if interleaved:
        return I.record(other=I.select(d < 2 * R, d + 1 - 2 * (d % 2), d), pair=I.minimum(d // 2, R - 1),
                        sign=I.select(d % 2 == 0, -1.0, 1.0), turned=d < 2 * R)
    return I.record(other=I.select(d < R, d + R, I.select(d < 2 * R, d - R, d)), pair=I.minimum(I.select(d < R, d, d - R), R - 1),
                    sign=I.select(d < R, -1.0, 1.0), turned=d < 2 * R)


@intent.fn
def rotate(y, cos, sin, interleaved, direction):
    """y [H, D] turned by one token's angles; direction -1 turns back."""
    at = rotation_partners(y.shape[1], cos.shape[0], interleaved)
    turned = y * cos[at.pair][None, :] + I.gather(y, index=(slice(None), at.other)) * (direction * at.sign * sin[at.pair])[None, :]
    return I.select(at.turned[None, :], turned, y)


@intent.fn
def norm_rotate(x, weight, cos, sin, eps, interleaved, element):
    rows = I.cast(x, I.f32)
    inverse = I.rsqrt(I.reduce.sum(rows * rows, axis=1) / x.shape[1] + eps)
    return I.cast(rotate(rows * inverse[:, None] * weight[None, :], cos, sin, interleaved, 1.0), element)


@intent.fn
def table_row(position, rows):
    return I.minimum(I.maximum(I.cast(position, I.index), 0), rows - 1)


@intent.kernel
def qk_norm_rope_f16(
    q: I.In[I.f16, ("T", "HQ", "D")],
    k: I.In[I.f16, ("T", "HK", "D")],
    q_weight: I.In[I.f32, ("D",)],
    k_weight: I.In[I.f32, ("D",)],
    positions: I.In[I.i32, ("T",)],
    cos: I.In[I.f32, ("P", "R")],
    sin: I.In[I.f32, ("P", "R")],
    q_output: I.Out[I.f16, ("T", "HQ", "D")],
    k_output: I.Out[I.f16, ("T", "HK", "D")],
    eps: I.f32,
    INTERLEAVED: I.Constexpr[bool],
):
    for t in I.parallel(I.domain(0, q.shape[0])):
        p = table_row(positions[t], cos.shape[0])
        q_output[t, :, :] = norm_rotate(q[t, :, :], q_weight, cos[p, :], sin[p, :], eps, INTERLEAVED, I.f16)
        k_output[t, :, :] = norm_rotate(k[t, :, :], k_weight, cos[p, :], sin[p, :], eps, INTERLEAVED, I.f16)


@intent.kernel
def qk_norm_rope_bf16(
    q: I.In[I.bf16, ("T", "HQ", "D")],
    k: I.In[I.bf16, ("T", "HK", "D")],
    q_weight: I.In[I.f32, ("D",)],
    k_weight: I.In[I.f32, ("D",)],
    positions: I.In[I.i32, ("T",)],
    cos: I.In[I.f32, ("P", "R")],
    sin: I.In[I.f32, ("P", "R")],
    q_output: I.Out[I.bf16, ("T", "HQ", "D")],
    k_output: I.Out[I.bf16, ("T", "HK", "D")],
    eps: I.f32,
    INTERLEAVED: I.Constexpr[bool],
):
    for t in I.parallel(I.domain(0, q.shape[0])):
        p = table_row(positions[t], cos.shape[0])
        q_output[t, :, :] = norm_rotate(q[t, :, :], q_weight, cos[p, :], sin[p, :], eps, INTERLEAVED, I.bf16)
        k_output[t, :, :] = norm_rotate(k[t, :, :], k_weight, cos[p, :], sin[p, :], eps, INTERLEAVED, I.bf16)
