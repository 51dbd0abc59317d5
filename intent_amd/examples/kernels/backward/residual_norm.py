"""Gradients of `residual_norm`: `residual_norm_backward_f16` and `residual_norm_backward_bf16`. No reference counterpart.

From the block's output x, the stored sum h, and the gradients that reach the sum and the output (gh, gy), with r_x, r_h = rsqrt(mean(..^2)
+ eps) formed again and u = x r_x wp (x where post_weight holds nothing):

  dh = gh + r_h (gy w - h r_h mean(gy w h r_h))
  grad_residual = residual_scale dh                       stored in the rows' type
  grad_gate = block_scale * sum of dh u                   a token's; nothing where gate holds nothing
  du = block_scale g dh
  grad_block = r_x (du wp - x r_x mean(du wp x r_x))      du where post_weight holds nothing; stored in the rows' type
  grad_post_weight = sum over tokens of du x r_x,  grad_weight = sum over tokens of gy h r_h       f32

The weights' sums run in a fixed order, so equal inputs give equal bits. A gradient of rows may be any of the rows that are read.
"""
import intent_amd as intent
import intent_amd.language as I


@intent.fn
def through_norm(row, weight, grad, eps):
    """What a norm passes on of its output's gradient, to its input and, of this row, to its weight."""
    inverse = I.rsqrt(I.reduce.sum(row * row, axis=0) / row.shape[0] + eps)
    unit, inner = row * inverse, grad * weight
    along = I.reduce.sum(inner * unit, axis=0) / row.shape[0]
    return I.record(row=inverse * (inner - unit * along), weight=grad * unit, output=unit * weight)


@intent.kernel
def residual_norm_backward_f16(
    block: I.In[I.f16, ("T", "D")],
    sum: I.In[I.f16, ("T", "D")],
    gate: I.In[I.f32, ("G",)],
    post_weight: I.In[I.f32, ("W",)],
    weight: I.In[I.f32, ("D",)],
    grad_sum: I.In[I.f16, ("T", "D")],
    grad_output: I.In[I.f16, ("T", "D")],
    grad_block: I.Out[I.f16, ("T", "D")],
    grad_residual: I.Out[I.f16, ("T", "D")],
    grad_gate: I.Out[I.f32, ("G",)],
    grad_post_weight: I.Out[I.f32, ("W",)],
    grad_weight: I.Out[I.f32, ("D",)],
    residual_scale: I.f32,
    block_scale: I.f32,
    eps: I.f32,
):
    grad_weight[:], grad_post_weight[:] = I.zeros(weight.shape, I.f32), I.zeros(post_weight.shape, I.f32)
    for t in I.domain(0, block.shape[0]):
        outer = through_norm(I.cast(sum[t, :], I.f32), weight[:], I.cast(grad_output[t, :], I.f32), eps)
        grad_weight[:] = grad_weight[:] + outer.weight
        grad = I.cast(grad_sum[t, :], I.f32) + outer.row
        grad_residual[t, :] = I.cast(residual_scale * grad, I.f16)
        branch = I.cast(block[t, :], I.f32)
        down = block_scale * grad
        if gate.shape[0] > 0:
            down = down * gate[t]
        if post_weight.shape[0] > 0:
            inner = through_norm(branch, post_weight[:], down, eps)
            branch, down = inner.output, inner.row
            grad_post_weight[:] = grad_post_weight[:] + inner.weight
        if gate.shape[0] > 0:
            grad_gate[t] = block_scale * I.reduce.sum(grad * branch, axis=0)
        grad_block[t, :] = I.cast(down, I.f16)


@intent.kernel
def residual_norm_backward_bf16(
    block: I.In[I.bf16, ("T", "D")],
    sum: I.In[I.bf16, ("T", "D")],
    gate: I.In[I.f32, ("G",)],
    post_weight: I.In[I.f32, ("W",)],
    weight: I.In[I.f32, ("D",)],
    grad_sum: I.In[I.bf16, ("T", "D")],
    grad_output: I.In[I.bf16, ("T", "D")],
    grad_block: I.Out[I.bf16, ("T", "D")],
    grad_residual: I.Out[I.bf16, ("T", "D")],
    grad_gate: I.Out[I.f32, ("G",)],
    grad_post_weight: I.Out[I.f32, ("W",)],
    grad_weight: I.Out[I.f32, ("D",)],
    residual_scale: I.f32,
    block_scale: I.f32,
    eps: I.f32,
):
    grad_weight[:], grad_post_weight[:] = I.zeros(weight.shape, I.f32), I.zeros(post_weight.shape, I.f32)
    for t in I.domain(0, block.shape[0]):
        outer = through_norm(I.cast(sum[t, :], I.f32), weight[:], I.cast(grad_output[t, :], I.f32), eps)
        grad_weight[:] = grad_weight[:] + outer.weight
        grad = I.cast(grad_sum[t, :], I.f32) + outer.row
        grad_residual[t, :] = I.cast(residual_scale * grad, I.bf16)
        branch = I.cast(block[t, :], I.f32)
        down = block_scale * grad
        if gate.shape[0] > 0:
            down = down * gate[t]
        if post_weight.shape[0] > 0:
            inner = through_norm(branch, post_weight[:], down, eps)
            branch, down = inner.output, inner.row
            grad_post_weight[:] = grad_post_weight[:] + inner.weight
        if gate.shape[0] > 0:
            grad_gate[t] = block_scale * I.reduce.sum(grad * branch, axis=0)
        grad_block[t, :] = I.cast(down, I.bf16)
