"""Attention of one new token per sequence of a batch that shares a prefix, which is read once for all, and of which each sequence has
tokens of its own: `paged_gqa_decode_prefix_f16` and `paged_gqa_decode_prefix_bf16`. No reference counterpart; the cache is that of
`paged_gqa_decode_partials`, pages of 16-bit rows.

The prefix is the first prefix_length[0] tokens of the pages prefix_indices, in order. Sequence s adds the first sequence_lengths[s]
tokens of the pages page_offsets[s] .. page_offsets[s + 1] of page_indices; its length does not count the prefix. Neither is more than its
pages hold. Query head h attends to key head h / HEAD_GROUP over both:

  output = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale * q . k_j - max)        0 where there is no token

Sums and weights are f32; weights enter the second product whole, as three numbers of the rows' type (but for 2^-36 of the largest in
f16). An infinite value gives an infinity, or NaN where its weight is below 2^-25 (f16) or 2^-126 (bf16) of the largest; a row all
of whose scores are -inf gives NaN. page_offsets start at 0 or above and do not decrease. Table entries outside their table and pages outside the cache read the nearest. Lengths, offsets and tables are read as they are
at the launch, so a captured graph follows them. D is 64 or 128.

The bodies state this one sequence at a time; the hip provider recognises a definition by name and signature.
"""
import intent_amd as intent
import intent_amd.language as I


@intent.fn
def token_rows(cache, indices, first, count, head):
    """Rows of `count` tokens of one head, from entry `first` of a page table on."""
    PS = cache.shape[1]
    token = I.indices(I.domain(0, count))
    entry = I.minimum(I.maximum(first + token // PS, 0), indices.shape[0] - 1)
    page = I.minimum(I.maximum(I.cast(indices[entry], I.index), 0), cache.shape[0] - 1)
    return cache[page, token % PS, head, :]


@intent.fn
def held(length, pages, cache):
    return I.minimum(I.maximum(I.cast(length, I.index), 0), I.maximum(pages, 0) * cache.shape[1])


@intent.fn
def shared_attention(queries, shared_keys, shared_values, keys, values, scale, element):
    """A group's rows over the prefix's tokens and a sequence's own."""
    old = I.matmul(queries, shared_keys, transpose_rhs=True, acc_dtype=I.f32) * scale
    new = I.matmul(queries, keys, transpose_rhs=True, acc_dtype=I.f32) * scale
    peak = I.maximum(I.reduce(old, axis=1, identity=-I.inf, combine=I.maximum_num),
                     I.reduce(new, axis=1, identity=-I.inf, combine=I.maximum_num))
    old, new = I.exp(old - peak[:, None]), I.exp(new - peak[:, None])
    total = I.reduce.sum(old, axis=1) + I.reduce.sum(new, axis=1)
    mixed = I.matmul(old, shared_values, acc_dtype=I.f32) + I.matmul(new, values, acc_dtype=I.f32)
    live = shared_keys.shape[0] + keys.shape[0] > 0
    return I.cast(I.select(live, mixed / total[:, None], 0.0), element)


@intent.kernel
def paged_gqa_decode_prefix_f16(
    q: I.In[I.f16, ("B", "HQ", "D")],
    key_cache: I.In[I.f16, ("P", "PS", "HK", "D")],
    value_cache: I.In[I.f16, ("P", "PS", "HK", "D")],
    prefix_indices: I.In[I.i32, ("S0",)],
    prefix_length: I.In[I.i32, ("ONE",)],
    page_offsets: I.In[I.i32, ("B_PLUS_1",)],
    page_indices: I.In[I.i32, ("S",)],
    sequence_lengths: I.In[I.i32, ("B",)],
    output: I.Out[I.f16, ("B", "HQ", "D")],
    scale: I.f32,
    HEAD_GROUP: I.Constexpr[int],
):
    prefix = held(prefix_length[0], prefix_indices.shape[0], key_cache)
    for s in I.parallel(I.domain(0, q.shape[0])):
        first = I.cast(page_offsets[s], I.index)
        own = held(sequence_lengths[s], I.cast(page_offsets[s + 1], I.index) - first, key_cache)
        for kv in I.parallel(I.domain(0, key_cache.shape[2])):
            heads = kv * HEAD_GROUP + I.indices(I.domain(0, HEAD_GROUP))
            result = shared_attention(
                I.gather(q, index=(s, heads, slice(None))), token_rows(key_cache, prefix_indices, 0, prefix, kv),
                token_rows(value_cache, prefix_indices, 0, prefix, kv), token_rows(key_cache, page_indices, first, own, kv),
                token_rows(value_cache, page_indices, first, own, kv), scale, I.f16)
            I.scatter_unique(output, index=(s, heads, slice(None)), value=result)


@intent.kernel
def paged_gqa_decode_prefix_bf16(
    q: I.In[I.bf16, ("B", "HQ", "D")],
    key_cache: I.In[I.bf16, ("P", "PS", "HK", "D")],
    value_cache: I.In[I.bf16, ("P", "PS", "HK", "D")],
    prefix_indices: I.In[I.i32, ("S0",)],
    prefix_length: I.In[I.i32, ("ONE",)],
    page_offsets: I.In[I.i32, ("B_PLUS_1",)],
    page_indices: I.In[I.i32, ("S",)],
    sequence_lengths: I.In[I.i32, ("B",)],
    output: I.Out[I.bf16, ("B", "HQ", "D")],
    scale: I.f32,
    HEAD_GROUP: I.Constexpr[int],
):
    prefix = held(prefix_length[0], prefix_indices.shape[0], key_cache)
    for s in I.parallel(I.domain(0, q.shape[0])):
        first = I.cast(page_offsets[s], I.index)
        own = held(sequence_lengths[s], I.cast(page_offsets[s + 1], I.index) - first, key_cache)
        for kv in I.parallel(I.domain(0, key_cache.shape[2])):
            heads = kv * HEAD_GROUP + I.indices(I.domain(0, HEAD_GROUP))
            result = shared_attention(
                I.gather(q, index=(s, heads, slice(None))), token_rows(key_cache, prefix_indices, 0, prefix, kv),
                token_rows(value_cache, prefix_indices, 0, prefix, kv), token_rows(key_cache, page_indices, first, own, kv),
                token_rows(value_cache, page_indices, first, own, kv), scale, I.bf16)
            I.scatter_unique(output, index=(s, heads, slice(None)), value=result)
