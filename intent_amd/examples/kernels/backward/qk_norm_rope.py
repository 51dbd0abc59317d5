"""Gradients of `qk_norm_rope`: `qk_norm_rope_backward_f16` and `qk_norm_rope_backward_bf16`. No reference counterpart.

With g the output's gradient turned back by the token's angles, r = rsqrt(mean(x^2) + eps) and u = x r (both formed again
from x, which is read anyway):

  grad_x = r (g w - u mean(g w u))             stored in the storage type
  grad_w = sum over tokens and heads of g u    f32

The weight's sums run in a fixed order, so equal inputs give equal bits.
"""
import intent_amd as intent
import intent_amd.language as I

from intent_amd.examples.kernels.normalization.qk_norm_rope import rotate, table_row


@intent.fn
def norm_rotate_backward(x, weight, grad, cos, sin, eps, interleaved, element):
    rows, g = I.cast(x, I.f32), rotate(I.cast(grad, I.f32), cos, sin, interleaved, -1.0)
    inverse = I.rsqrt(I.reduce.sum(rows * rows, axis=1) / x.shape[1] + eps)
    unit, inner = rows * inverse[:, None], g * weight[None, :]
    along = I.reduce.sum(inner * unit, axis=1) / x.shape[1]
    return I.record(x=I.cast(inverse[:, None] * (inner - unit * along[:, None]), element), weight=I.reduce.sum(g * unit, axis=0))


@intent.kernel
def qk_norm_rope_backward_f16(
    q: I.In[I.f16, ("T", "HQ", "D")],
    k: I.In[I.f16, ("T", "HK", "D")],
    q_weight: I.In[I.f32, ("D",)],
    k_weight: I.In[I.f32, ("D",)],
    positions: I.In[I.i32, ("T",)],
    cos: I.In[I.f32, ("P", "R")],
    sin: I.In[I.f32, ("P", "R")],
    grad_q_output: I.In[I.f16, ("T", "HQ", "D")],
    grad_k_output: I.In[I.f16, ("T", "HK", "D")],
    grad_q: I.Out[I.f16, ("T", "HQ", "D")],
    grad_k: I.Out[I.f16, ("T", "HK", "D")],
    grad_q_weight: I.Out[I.f32, ("D",)],
    grad_k_weight: I.Out[I.f32, ("D",)],
    eps: I.f32,
    INTERLEAVED: I.Constexpr[bool],
):
    grad_q_weight[:], grad_k_weight[:] = I.zeros(q.shape[2:], I.f32), I.zeros(q.shape[2:], I.f32)
    for t in I.domain(0, q.shape[0]):
        p = table_row(positions[t], cos.shape[0])
        dq = norm_rotate_backward(q[t, :, :], q_weight, grad_q_output[t, :, :], cos[p, :], sin[p, :], eps, INTERLEAVED, I.f16)
        dk = norm_rotate_backward(k[t, :, :], k_weight, grad_k_output[t, :, :], cos[p, :], sin[p, :], eps, INTERLEAVED, I.f16)
        grad_q[t, :, :], grad_k[t, :, :] = dq.x, dk.x
        grad_q_weight[:], grad_k_weight[:] = grad_q_weight[:] + dq.weight, grad_k_weight[:] + dk.weight


@intent.kernel
def qk_norm_rope_backward_bf16(
    q: I.In[I.bf16, ("T", "HQ", "D")],
    k: I.In[I.bf16, ("T", "HK", "D")],
    q_weight: I.In[I.f32, ("D",)],
    k_weight: I.In[I.f32, ("D",)],
    positions: I.In[I.i32, ("T",)],
    cos: I.In[I.f32, ("P", "R")],
    sin: I.In[I.f32, ("P", "R")],
    grad_q_output: I.In[I.bf16, ("T", "HQ", "D")],
    grad_k_output: I.In[I.bf16, ("T", "HK", "D")],
    grad_q: I.Out[I.bf16, ("T", "HQ", "D")],
    grad_k: I.Out[I.bf16, ("T", "HK", "D")],
    grad_q_weight: I.Out[I.f32, ("D",)],
    grad_k_weight: I.Out[I.f32, ("D",)],
    eps: I.f32,
    INTERLEAVED: I.Constexpr[bool],
):
    grad_q_weight[:], grad_k_weight[:] = I.zeros(q.shape[2:], I.f32), I.zeros(q.shape[2:], I.f32)
    for t in I.domain(0, q.shape[0]):
        p = table_row(positions[t], cos.shape[0])
        dq = norm_rotate_backward(q[t, :, :], q_weight, grad_q_output[t, :, :], cos[p, :], sin[p, :], eps, INTERLEAVED, I.bf16)
        dk = norm_rotate_backward(k[t, :, :], k_weight, grad_k_output[t, :, :], cos[p, :], sin[p, :], eps, INTERLEAVED, I.bf16)
        grad_q[t, :, :], grad_k[t, :, :] = dq.x, dk.x
        grad_q_weight[:], grad_k_weight[:] = grad_q_weight[:] + dq.weight, grad_k_weight[:] + dk.weight
