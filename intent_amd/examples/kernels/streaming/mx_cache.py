"""A paged key-value cache of 8 bits a value: rows written into it (`paged_cache_append_*`), read back
(`paged_cache_read_*`), and the attention of one new token over it (`paged_gqa_decode_mx_*`), each for f16 and bf16 rows.
No reference counterpart; the tables are those of `paged_gqa_decode_partials` (streaming/paged_attention.py).

Cache. Elements f8e4m3fn [P, PS, HK, D] and exponents u8 [P, PS, HK, D / 32]: element i of a row stands for
element * 2^(exponent[i / 32] - 127); exponent 255 stands for NaN. Any order of the page, token and head axes may lie in
memory (a [P, HK, PS, D] allocation seen through a transpose keeps a head's page together), and keys and values may be slices
of one allocation ([P, 2, PS, HK, D]). Sequence s holds the logical
pages page_offsets[s] .. page_offsets[s + 1] of page_indices; its position p is place p % PS of logical page p / PS. A page
that several sequences name may be read by all and appended to by one.

Writing. A block of 32 takes the smallest exponent e >= -127 with max |x| <= 448 * 2^e over its finite values, and each
element is e4m3(x * 2^-e), rounded to nearest even. NaN and infinities are held as NaN (e4m3 has no infinity).

Reading. A value is element * 2^e rounded to the row type: exact, apart from f16's subnormals and largest values.

The bodies state this densely, one row or sequence at a time; the hip provider recognises a definition by name and
signature.
"""
import intent_amd as intent
import intent_amd.language as I

from intent_amd.examples.kernels.streaming.attention import causal_pairs

BLOCK = 32
LARGEST = 448.0


@intent.fn
def quantise(row, blocks):
    """A row's elements and exponent bytes."""
    values = I.reshape(I.cast(row, I.f32), (blocks, BLOCK))
    finite = I.abs(values) < I.inf
    size = I.reduce(I.select(finite, I.abs(values), 0.0), axis=1, identity=0.0, combine=I.maximum)
    exponent = I.maximum(I.select(size > 0.0, power_above(size / LARGEST), -127), -127)
    elements = I.cast(I.select(finite, values * I.exp2(-exponent)[:, None], I.inf - I.inf), I.f8e4m3fn)
    return I.record(elements=I.reshape(elements, (blocks * BLOCK,)), exponents=I.cast(exponent + 127, I.u8))


@intent.fn
def power_above(x):
    """The smallest integer e with x <= 2^e (exactly; the logarithm's rounding settled by a comparison)."""
    e = I.floor(I.log(x) * I.LOG2E)
    return I.select(x > I.exp2(e + 1.0), e + 2, I.select(x > I.exp2(e), e + 1, e))


@intent.fn
def dequantise(elements, exponents, element):
    rows = I.reshape(I.cast(elements, I.f32), (elements.shape[0], exponents.shape[1], BLOCK))
    return I.cast(I.reshape(rows * I.exp2(I.cast(exponents, I.f32) - 127.0)[:, :, None], elements.shape), element)


@intent.fn
def slot_of(page_offsets, page_indices, s, position, PS):
    """Page and place of positions of sequence s, and whether the tables have them."""
    first = I.cast(page_offsets[s], I.index)
    at = position // PS
    inside = (position >= 0) & (first + at < I.cast(page_offsets[s + 1], I.index))
    return I.record(page=I.cast(page_indices[I.select(inside, first + at, 0)], I.index), place=position % PS, inside=inside)


@intent.fn
def append_rows(rows, cache, exponents, cu_seqlens, page_offsets, page_indices, sequence_lengths):
    for s in I.parallel(I.domain(0, sequence_lengths.shape[0])):
        first, last = I.cast(cu_seqlens[s], I.index), I.cast(cu_seqlens[s + 1], I.index)
        for row in I.parallel(I.domain(first, last)):
            position = I.cast(sequence_lengths[s], I.index) - (last - row)
            slot = slot_of(page_offsets, page_indices, s, position, cache.shape[1])
            if slot.inside & (slot.page >= 0) & (slot.page < cache.shape[0]):
                for h in I.parallel(I.domain(0, rows.shape[1])):
                    held = quantise(rows[row, h, :], exponents.shape[3])
                    cache[slot.page, slot.place, h, :] = held.elements
                    exponents[slot.page, slot.place, h, :] = held.exponents


@intent.fn
def read_rows(cache, exponents, cu_seqlens, page_offsets, page_indices, out, element):
    for s in I.parallel(I.domain(0, cu_seqlens.shape[0] - 1)):
        first, last = I.cast(cu_seqlens[s], I.index), I.cast(cu_seqlens[s + 1], I.index)
        for row in I.parallel(I.domain(first, last)):
            slot = slot_of(page_offsets, page_indices, s, row - first, cache.shape[1])
            inside = slot.inside & (slot.page >= 0) & (slot.page < cache.shape[0])
            held = dequantise(cache[slot.page, slot.place, :, :], exponents[slot.page, slot.place, :, :], element)
            out[row, :, :] = I.select(inside, held, 0.0)


@intent.kernel
def paged_cache_append_f16(
    k: I.In[I.f16, ("U", "HK", "D")],
    v: I.In[I.f16, ("U", "HK", "DV")],
    key_cache: I.InOut[I.f8e4m3fn, ("P", "PS", "HK", "D")],
    key_exponents: I.InOut[I.u8, ("P", "PS", "HK", "DB")],
    value_cache: I.InOut[I.f8e4m3fn, ("P", "PS", "HK", "DV")],
    value_exponents: I.InOut[I.u8, ("P", "PS", "HK", "DVB")],
    cu_seqlens: I.In[I.i32, ("B_PLUS_1",)],
    page_offsets: I.In[I.i32, ("B_PLUS_1",)],
    page_indices: I.In[I.i32, ("S",)],
    sequence_lengths: I.In[I.i32, ("B",)],
):
    """Rows cu_seqlens[s] .. cu_seqlens[s + 1] of k and v become the last positions of sequence s, whose length with them is
    sequence_lengths[s]. Rows behind the last sequence and positions that the tables have no page for are left out."""
    append_rows(k, key_cache, key_exponents, cu_seqlens, page_offsets, page_indices, sequence_lengths)
    append_rows(v, value_cache, value_exponents, cu_seqlens, page_offsets, page_indices, sequence_lengths)


@intent.kernel
def paged_cache_append_bf16(
    k: I.In[I.bf16, ("U", "HK", "D")],
    v: I.In[I.bf16, ("U", "HK", "DV")],
    key_cache: I.InOut[I.f8e4m3fn, ("P", "PS", "HK", "D")],
    key_exponents: I.InOut[I.u8, ("P", "PS", "HK", "DB")],
    value_cache: I.InOut[I.f8e4m3fn, ("P", "PS", "HK", "DV")],
    value_exponents: I.InOut[I.u8, ("P", "PS", "HK", "DVB")],
    cu_seqlens: I.In[I.i32, ("B_PLUS_1",)],
    page_offsets: I.In[I.i32, ("B_PLUS_1",)],
    page_indices: I.In[I.i32, ("S",)],
    sequence_lengths: I.In[I.i32, ("B",)],
):
    append_rows(k, key_cache, key_exponents, cu_seqlens, page_offsets, page_indices, sequence_lengths)
    append_rows(v, value_cache, value_exponents, cu_seqlens, page_offsets, page_indices, sequence_lengths)


@intent.kernel
def paged_cache_read_f16(
    key_cache: I.In[I.f8e4m3fn, ("P", "PS", "HK", "D")],
    key_exponents: I.In[I.u8, ("P", "PS", "HK", "DB")],
    value_cache: I.In[I.f8e4m3fn, ("P", "PS", "HK", "DV")],
    value_exponents: I.In[I.u8, ("P", "PS", "HK", "DVB")],
    cu_seqlens: I.In[I.i32, ("B_PLUS_1",)],
    page_offsets: I.In[I.i32, ("B_PLUS_1",)],
    page_indices: I.In[I.i32, ("S",)],
    k: I.Out[I.f16, ("U", "HK", "D")],
    v: I.Out[I.f16, ("U", "HK", "DV")],
):
    """Row cu_seqlens[s] + i of k and v is position i of sequence s, 0 where the tables have no page for it. Rows behind the
    last sequence keep what they held. The caller gives the outputs (how many rows there are stands on the device)."""
    read_rows(key_cache, key_exponents, cu_seqlens, page_offsets, page_indices, k, I.f16)
    read_rows(value_cache, value_exponents, cu_seqlens, page_offsets, page_indices, v, I.f16)


@intent.kernel
def paged_cache_read_bf16(
    key_cache: I.In[I.f8e4m3fn, ("P", "PS", "HK", "D")],
    key_exponents: I.In[I.u8, ("P", "PS", "HK", "DB")],
    value_cache: I.In[I.f8e4m3fn, ("P", "PS", "HK", "DV")],
    value_exponents: I.In[I.u8, ("P", "PS", "HK", "DVB")],
    cu_seqlens: I.In[I.i32, ("B_PLUS_1",)],
    page_offsets: I.In[I.i32, ("B_PLUS_1",)],
    page_indices: I.In[I.i32, ("S",)],
    k: I.Out[I.bf16, ("U", "HK", "D")],
    v: I.Out[I.bf16, ("U", "HK", "DV")],
):
    read_rows(key_cache, key_exponents, cu_seqlens, page_offsets, page_indices, k, I.bf16)
    read_rows(value_cache, value_exponents, cu_seqlens, page_offsets, page_indices, v, I.bf16)


@intent.fn
def decode_head(query, k_rows, v_rows, scale, element):
    """One query head over its sequence's rows: f32 throughout, rounded at the end; 0 where there is no row."""
    logits = I.matmul(query, k_rows, transpose_rhs=True, acc_dtype=I.f32) * (scale * I.LOG2E)
    live = I.reduce.any(causal_pairs(I.indices(I.domain(0, 1)), I.indices(I.domain(0, k_rows.shape[0])), False), axis=1)
    peak = I.reduce(logits, axis=1, identity=-I.inf, combine=I.maximum_num)
    weights = I.exp2(logits - peak[:, None], approximate=True, flush_to_zero=True)
    mixed = I.matmul(weights, I.cast(v_rows, I.f32), acc_dtype=I.f32)
    return I.cast(I.select(live[:, None], mixed / I.reduce.sum(weights, axis=1)[:, None], 0.0), element)


@intent.fn
def decode_rows(q, key_cache, key_exponents, value_cache, value_exponents, page_offsets, page_indices, sequence_lengths, output,
                scale, group, element):
    P, PS = key_cache.shape[0], key_cache.shape[1]
    for s in I.parallel(I.domain(0, q.shape[0])):
        held = (I.cast(page_offsets[s + 1], I.index) - I.cast(page_offsets[s], I.index)) * PS
        position = I.indices(I.domain(0, I.minimum(I.cast(sequence_lengths[s], I.index), held)))
        slot = slot_of(page_offsets, page_indices, s, position, PS)
        place = I.members(slot, (slot.page >= 0) & (slot.page < P))
        for h in I.parallel(I.domain(0, q.shape[1])):
            shared = h // group
            keys = dequantise(key_cache[place.page, place.place, shared, :], key_exponents[place.page, place.place, shared, :], element)
            values = dequantise(value_cache[place.page, place.place, shared, :], value_exponents[place.page, place.place, shared, :],
                                element)
            output[s, h, :] = decode_head(I.reshape(q[s, h, :], (1, q.shape[2])), keys, values, scale, element)[0]


@intent.kernel
def paged_gqa_decode_mx_f16(
    q: I.In[I.f16, ("B", "HQ", "D")],
    key_cache: I.In[I.f8e4m3fn, ("P", "PS", "HK", "D")],
    key_exponents: I.In[I.u8, ("P", "PS", "HK", "DB")],
    value_cache: I.In[I.f8e4m3fn, ("P", "PS", "HK", "D")],
    value_exponents: I.In[I.u8, ("P", "PS", "HK", "DB")],
    page_offsets: I.In[I.i32, ("B_PLUS_1",)],
    page_indices: I.In[I.i32, ("S",)],
    sequence_lengths: I.In[I.i32, ("B",)],
    output: I.Out[I.f16, ("B", "HQ", "D")],
    scale: I.f32,
    HEAD_GROUP: I.Constexpr[int],
):
    """Query head h of sequence s over the positions below sequence_lengths[s] that the tables have a page for, with the keys
    and values of head h // HEAD_GROUP; 0 where there is none. page_offsets do not decrease; pages reserved beyond a
    sequence's length are not read. D is 64, 96, 128, 192 or 256. Any head group; the work is cut over each sequence's
    pages and joined within the call."""
    decode_rows(q, key_cache, key_exponents, value_cache, value_exponents, page_offsets, page_indices, sequence_lengths, output,
                scale, HEAD_GROUP, I.f16)


@intent.kernel
def paged_gqa_decode_mx_bf16(
    q: I.In[I.bf16, ("B", "HQ", "D")],
    key_cache: I.In[I.f8e4m3fn, ("P", "PS", "HK", "D")],
    key_exponents: I.In[I.u8, ("P", "PS", "HK", "DB")],
    value_cache: I.In[I.f8e4m3fn, ("P", "PS", "HK", "D")],
    value_exponents: I.In[I.u8, ("P", "PS", "HK", "DB")],
    page_offsets: I.In[I.i32, ("B_PLUS_1",)],
    page_indices: I.In[I.i32, ("S",)],
    sequence_lengths: I.In[I.i32, ("B",)],
    output: I.Out[I.bf16, ("B", "HQ", "D")],
    scale: I.f32,
    HEAD_GROUP: I.Constexpr[int],
):
    decode_rows(q, key_cache, key_exponents, value_cache, value_exponents, page_offsets, page_indices, sequence_lengths, output,
                scale, HEAD_GROUP, I.bf16)
