"""The residual stream after a block's output has joined it, and its norm, in one pass over the rows: `residual_norm_f16` and
`residual_norm_bf16`, and with the norm in 8 bits `residual_norm_i8_f16` and `residual_norm_i8_bf16`. No reference counterpart.

For a token's row x of the block's output and s of the stream, of width D, its gate g, weights wp (of the block's own norm) and w:

  u = x * rsqrt(mean(x^2) + eps) * wp                     u = x where post_weight holds nothing
  h = residual_scale * s + block_scale * g * u            f32; sum = h in the rows' type; g = 1 where gate holds nothing
  y = h * rsqrt(mean(h^2) + eps) * w                      output = y in the rows' type

or, in 8 bits, output = round(127 y / max|y|), halves to even, and scales = max|y| / 127: y is about output * scale. A row of zeros
has a scale of 0; one with an infinity or NaN a scale of NaN and elements of 0. Norms are formed from h before it is rounded.

D is at most 16384. `sum` may be `residual` or `block` itself, and so may `output` where it is not 8 bits.

The bodies state this one token at a time; the hip provider recognises a definition by name and signature.
"""
import intent_amd as intent
import intent_amd.language as I

from intent_amd.examples.kernels.normalization.quantize_rows import quantised


@intent.fn
def root_mean_square_norm(row, weight, eps):
    return row * I.rsqrt(I.reduce.sum(row * row, axis=0) / row.shape[0] + eps) * weight


@intent.fn
def joined(block, residual, gate, post_weight, token, residual_scale, block_scale, eps):
    """The stream's row of a token behind the block, in f32."""
    branch = I.cast(block, I.f32)
    if post_weight.shape[0] > 0:
        branch = root_mean_square_norm(branch, post_weight[:], eps)
    if gate.shape[0] > 0:
        branch = branch * gate[token]
    return I.cast(residual, I.f32) * residual_scale + branch * block_scale


@intent.kernel
def residual_norm_f16(
    block: I.In[I.f16, ("T", "D")],
    residual: I.In[I.f16, ("T", "D")],
    gate: I.In[I.f32, ("G",)],
    post_weight: I.In[I.f32, ("W",)],
    weight: I.In[I.f32, ("D",)],
    sum: I.Out[I.f16, ("T", "D")],
    output: I.Out[I.f16, ("T", "D")],
    residual_scale: I.f32,
    block_scale: I.f32,
    eps: I.f32,
):
    for t in I.parallel(I.domain(0, block.shape[0])):
        h = joined(block[t, :], residual[t, :], gate, post_weight, t, residual_scale, block_scale, eps)
        sum[t, :] = I.cast(h, I.f16)
        output[t, :] = I.cast(root_mean_square_norm(h, weight[:], eps), I.f16)


@intent.kernel
def residual_norm_bf16(
    block: I.In[I.bf16, ("T", "D")],
    residual: I.In[I.bf16, ("T", "D")],
    gate: I.In[I.f32, ("G",)],
    post_weight: I.In[I.f32, ("W",)],
    weight: I.In[I.f32, ("D",)],
    sum: I.Out[I.bf16, ("T", "D")],
    output: I.Out[I.bf16, ("T", "D")],
    residual_scale: I.f32,
    block_scale: I.f32,
    eps: I.f32,
):
    for t in I.parallel(I.domain(0, block.shape[0])):
        h = joined(block[t, :], residual[t, :], gate, post_weight, t, residual_scale, block_scale, eps)
        sum[t, :] = I.cast(h, I.bf16)
        output[t, :] = I.cast(root_mean_square_norm(h, weight[:], eps), I.bf16)


@intent.kernel
def residual_norm_i8_f16(
    block: I.In[I.f16, ("T", "D")],
    residual: I.In[I.f16, ("T", "D")],
    gate: I.In[I.f32, ("G",)],
    post_weight: I.In[I.f32, ("W",)],
    weight: I.In[I.f32, ("D",)],
    sum: I.Out[I.f16, ("T", "D")],
    output: I.Out[I.i8, ("T", "D")],
    scales: I.Out[I.f32, ("T",)],
    residual_scale: I.f32,
    block_scale: I.f32,
    eps: I.f32,
):
    for t in I.parallel(I.domain(0, block.shape[0])):
        h = joined(block[t, :], residual[t, :], gate, post_weight, t, residual_scale, block_scale, eps)
        sum[t, :] = I.cast(h, I.f16)
        row = quantised(root_mean_square_norm(h, weight[:], eps))
        output[t, :], scales[t] = row.elements, row.scale


@intent.kernel
def residual_norm_i8_bf16(
    block: I.In[I.bf16, ("T", "D")],
    residual: I.In[I.bf16, ("T", "D")],
    gate: I.In[I.f32, ("G",)],
    post_weight: I.In[I.f32, ("W",)],
    weight: I.In[I.f32, ("D",)],
    sum: I.Out[I.bf16, ("T", "D")],
    output: I.Out[I.i8, ("T", "D")],
    scales: I.Out[I.f32, ("T",)],
    residual_scale: I.f32,
    block_scale: I.f32,
    eps: I.f32,
):
    for t in I.parallel(I.domain(0, block.shape[0])):
        h = joined(block[t, :], residual[t, :], gate, post_weight, t, residual_scale, block_scale, eps)
        sum[t, :] = I.cast(h, I.bf16)
        row = quantised(root_mean_square_norm(h, weight[:], eps))
        output[t, :], scales[t] = row.elements, row.scale
