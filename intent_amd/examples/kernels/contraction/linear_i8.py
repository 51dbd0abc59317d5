"""Products of 8-bit integers with a scale for each row of x (a token) and each row of the weight (a channel): `linear_i8_f16` and
`linear_i8_bf16`. No reference counterpart; the layout is that of `linear_f32` (weight rows [N, K]), the rows those of `quantize_rows`.

  y[m, n] = (sum_k x[m, k] weight[n, k]) * x_scales[m] * weight_scales[n] + bias[n]

The sums are int32 and exact: K is below 131072, and a multiple of 16. The rest is f32, rounded once to the output's type. `bias` holds N
numbers, or none. M and N are free.

The bodies state this densely; the hip provider recognises a definition by name and signature.
"""
import intent_amd as intent
import intent_amd.language as I


@intent.kernel
def linear_i8_f16(
    x: I.In[I.i8, ("M", "K")],
    weight: I.In[I.i8, ("N", "K")],
    x_scales: I.In[I.f32, ("M",)],
    weight_scales: I.In[I.f32, ("N",)],
    bias: I.In[I.f32, ("B",)],
    output: I.Out[I.f16, ("M", "N")],
):
    whole = I.cast(I.matmul(x[:, :], weight[:, :], transpose_rhs=True, acc_dtype=I.i32), I.f32)
    scaled = whole * x_scales[:][:, None] * weight_scales[:][None, :]
    if bias.shape[0] > 0:
        scaled = scaled + bias[:][None, :]
    output[:, :] = I.cast(scaled, I.f16)


@intent.kernel
def linear_i8_bf16(
    x: I.In[I.i8, ("M", "K")],
    weight: I.In[I.i8, ("N", "K")],
    x_scales: I.In[I.f32, ("M",)],
    weight_scales: I.In[I.f32, ("N",)],
    bias: I.In[I.f32, ("B",)],
    output: I.Out[I.bf16, ("M", "N")],
):
    whole = I.cast(I.matmul(x[:, :], weight[:, :], transpose_rhs=True, acc_dtype=I.i32), I.f32)
    scaled = whole * x_scales[:][:, None] * weight_scales[:][None, :]
    if bias.shape[0] > 0:
        scaled = scaled + bias[:][None, :]
    output[:, :] = I.cast(scaled, I.bf16)
