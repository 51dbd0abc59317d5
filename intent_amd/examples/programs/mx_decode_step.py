"""The attention of a layer for one new token per sequence, over a paged cache of 8 bits and with 4-bit weights, as one
prepared program: `MxDecodeStep`. No reference counterpart.

A prepared step binds, in launch order:

1. `linear_mxfp4_*`: the rows' queries, keys and values, [B, (HQ + 2 HK) D];
2. `qk_norm_rope_*` over the query and key slices of 1, in place of a copy;
3. `paged_cache_append_*`: the turned keys of 2 and the values of 1 become each sequence's last position;
4. `paged_gqa_decode_mx_*` over the cache with them;
5. `linear_mxfp4_*`: the heads of 4 to the layer's output [B, hidden].

The step reads `x`, `positions`, `sequence_lengths` and the tables as they are at the launch, so a serving loop writes the next
token's into them and launches again, or replays a graph that captured the launch. A sequence without pages (an idle place
of the batch) writes nothing into the cache; its heads are 0.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import ClassVar

from intent_amd.examples.kernels.contraction import linear_mxfp4
from intent_amd.examples.kernels.normalization import qk_norm_rope
from intent_amd.examples.kernels.streaming import mx_cache
from intent_amd.runtime import PreparedSequence


@dataclass(frozen=True)
class MxDecodeStep:
    mutable_inputs: ClassVar[tuple[int, ...]] = (10, 11, 12, 13)     # the cache
    project: object          # JIT kernel of linear_mxfp4
    turn: object             # JIT kernel of qk_norm_rope
    append: object           # JIT kernel of paged_cache_append
    attend: object           # JIT kernel of paged_gqa_decode_mx

    @classmethod
    def from_jit(cls, jit, *, dtype, head_group, interleaved=False):
        """Jit the kernels for rows of `dtype` ("f16" or "bf16") through `jit`."""
        return cls(project=jit(getattr(linear_mxfp4, f"linear_mxfp4_{dtype}")),
                   turn=jit(getattr(qk_norm_rope, f"qk_norm_rope_{dtype}"), constexprs=dict(INTERLEAVED=interleaved)),
                   append=jit(getattr(mx_cache, f"paged_cache_append_{dtype}")),
                   attend=jit(getattr(mx_cache, f"paged_gqa_decode_mx_{dtype}"), constexprs=dict(HEAD_GROUP=head_group)))

    def prepare(self, x, qkv_weight, qkv_exponents, out_weight, out_exponents, q_weight, k_weight, positions, cos, sin,
                key_cache, key_exponents, value_cache, value_exponents, cu_seqlens, page_offsets, page_indices,
                sequence_lengths, eps, scale, *, output=None):
        """`cu_seqlens` is 0, 1 .. B: a new row per sequence. `positions` are the new tokens' (sequence_lengths - 1, unless the
        caller counts otherwise) and `sequence_lengths` count them."""
        kv_heads, d = key_cache.shape[2:]
        cache = (key_cache, key_exponents, value_cache, value_exponents)
        project = self.project.prepare(x, qkv_weight, qkv_exponents)
        heads = project.result().unflatten(1, (-1, d))
        q_heads = heads.shape[1] - 2 * kv_heads
        q, k, v = heads.split((q_heads, kv_heads, kv_heads), 1)
        turn = self.turn.prepare(q, k, q_weight, k_weight, positions, cos, sin, eps)
        q, k = turn.result()
        append = self.append.prepare(k, v, *cache, cu_seqlens, page_offsets, page_indices, sequence_lengths)
        attend = self.attend.prepare(q, *cache, page_offsets, page_indices, sequence_lengths, scale)
        back = self.project.prepare(attend.result().flatten(1), out_weight, out_exponents,
                                    outputs=None if output is None else (output,))
        return PreparedSequence((project, turn, append, attend, back), outputs=back.result())

    def run(self, *arguments, **bindings):
        prepared = self.prepare(*arguments, **bindings)
        prepared.launch()
        return prepared.result()
