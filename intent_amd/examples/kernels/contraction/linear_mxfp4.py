"""Products with 4-bit weights that share a power of two per 32 along K (the OCP MXFP4 format): `linear_mxfp4_f16` and
`linear_mxfp4_bf16`. No reference counterpart; the layout is that of `linear_f32` (weight rows [N, K]).

weight u8 [N, K / 2] holds two e2m1 elements a byte, the even column in the low four bits (sign, two exponent bits, one
fraction bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6); exponents u8 [N, K / 32], 255 standing for NaN:

  W[n, k] = element * 2^(exponents[n, k / 32] - 127), in the type of x    exact, apart from f16's subnormals and largest values
  y[m, n] = sum_k x[m, k] W[n, k]                                         f32, stored in the type of x

K is a multiple of 32; M and N are free. The bodies state this densely; the hip provider recognises a definition by name and
signature.
"""
import intent_amd as intent
import intent_amd.language as I

BLOCK = 32


@intent.fn
def unpack(weight, exponents, element):
    """Rows of packed elements and their exponents as values of `element`."""
    N, half = weight.shape
    code = I.reshape(I.join(weight % 16, weight // 16), (N, 2 * half))          # the low four bits first
    power, fraction = code // 2 % 4, I.cast(code % 2, I.f32)
    size = I.select(power == 0, 0.5 * fraction, (1.0 + 0.5 * fraction) * I.exp2(I.cast(power, I.f32) - 1.0))
    signed = I.reshape(I.select(code >= 8, -size, size), (N, exponents.shape[1], BLOCK))
    scaled = signed * I.exp2(I.cast(exponents, I.f32) - 127.0)[:, :, None]
    return I.cast(I.reshape(scaled, (N, 2 * half)), element)


@intent.kernel
def linear_mxfp4_f16(
    x: I.In[I.f16, ("M", "K")],
    weight: I.In[I.u8, ("N", "K2")],
    exponents: I.In[I.u8, ("N", "KB")],
    output: I.Out[I.f16, ("M", "N")],
):
    values = unpack(weight[:, :], exponents[:, :], I.f16)
    output[:, :] = I.cast(I.matmul(x[:, :], values, transpose_rhs=True, acc_dtype=I.f32), I.f16)


@intent.kernel
def linear_mxfp4_bf16(
    x: I.In[I.bf16, ("M", "K")],
    weight: I.In[I.u8, ("N", "K2")],
    exponents: I.In[I.u8, ("N", "KB")],
    output: I.Out[I.bf16, ("M", "N")],
):
    values = unpack(weight[:, :], exponents[:, :], I.bf16)
    output[:, :] = I.cast(I.matmul(x[:, :], values, transpose_rhs=True, acc_dtype=I.f32), I.bf16)
