"""Rows made 8-bit integers with a scale each, the operands of `linear_i8`: `quantize_rows_f16`, `quantize_rows_bf16`, and of the gated
product of a feed-forward block `swiglu_quantize_rows_f16`, `swiglu_quantize_rows_bf16`. No reference counterpart.

For a row a (x, or gate * sigmoid(gate) * up in f32), of at most 32768 elements:

  scales = max|a| / 127,  output = round(127 a / max|a|), halves to even

so a is about output * scale. A row of zeros has a scale of 0; one with an infinity or NaN a scale of NaN and elements of 0. `gate` and
`up` may be halves of one projection's rows.

The bodies state this one row at a time; the hip provider recognises a definition by name and signature.
"""
import intent_amd as intent
import intent_amd.language as I


@intent.fn
def nearest(x):
    """x rounded to a whole number, halves to even (|x| below 2^22)."""
    return (x + 12582912.0) - 12582912.0


@intent.fn
def quantised(row):
    most = I.reduce(I.abs(row), axis=0, identity=0.0, combine=I.maximum)
    finite = most < I.inf
    quotient = row * 127.0 / I.select(most > 0.0, most, 1.0)
    return I.record(elements=I.cast(I.select(finite, nearest(quotient), 0.0), I.i8), scale=I.select(finite, most / 127.0, I.inf - I.inf))


@intent.kernel
def quantize_rows_f16(
    x: I.In[I.f16, ("M", "K")],
    output: I.Out[I.i8, ("M", "K")],
    scales: I.Out[I.f32, ("M",)],
):
    for m in I.parallel(I.domain(0, x.shape[0])):
        row = quantised(I.cast(x[m, :], I.f32))
        output[m, :], scales[m] = row.elements, row.scale


@intent.kernel
def quantize_rows_bf16(
    x: I.In[I.bf16, ("M", "K")],
    output: I.Out[I.i8, ("M", "K")],
    scales: I.Out[I.f32, ("M",)],
):
    for m in I.parallel(I.domain(0, x.shape[0])):
        row = quantised(I.cast(x[m, :], I.f32))
        output[m, :], scales[m] = row.elements, row.scale


@intent.kernel
def swiglu_quantize_rows_f16(
    gate: I.In[I.f16, ("M", "K")],
    up: I.In[I.f16, ("M", "K")],
    output: I.Out[I.i8, ("M", "K")],
    scales: I.Out[I.f32, ("M",)],
):
    for m in I.parallel(I.domain(0, gate.shape[0])):
        g = I.cast(gate[m, :], I.f32)
        row = quantised(g * I.sigmoid(g) * I.cast(up[m, :], I.f32))
        output[m, :], scales[m] = row.elements, row.scale


@intent.kernel
def swiglu_quantize_rows_bf16(
    gate: I.In[I.bf16, ("M", "K")],
    up: I.In[I.bf16, ("M", "K")],
    output: I.Out[I.i8, ("M", "K")],
    scales: I.Out[I.f32, ("M",)],
):
    for m in I.parallel(I.domain(0, gate.shape[0])):
        g = I.cast(gate[m, :], I.f32)
        row = quantised(g * I.sigmoid(g) * I.cast(up[m, :], I.f32))
        output[m, :], scales[m] = row.elements, row.scale
