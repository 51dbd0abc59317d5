"""The rest of a decoder layer behind its cache, for one new token per sequence of a batch that shares a prefix and with products of 8-bit
integers, as one prepared program: `Int8LayerStep`. No reference counterpart.

A prepared step binds, in launch order:

1. `paged_gqa_decode_prefix_*`: the heads' attention, [B, HQ, D];
2. `quantize_rows_*`, `linear_i8_*`: its projection to the stream's width, [B, hidden];
3. `residual_norm_i8_*`: the stream with it, and the feed-forward block's input in 8 bits;
4. `linear_i8_*`: the block's gate and up halves, [B, 2 F];
5. `swiglu_quantize_rows_*`, `linear_i8_*`: their gated product and the way back, [B, hidden];
6. `residual_norm_*`: the stream behind the layer, and the next layer's input.

A weight is (rows [N, K] of 8-bit integers, their scales [N], bias [N] or of no number). The step reads `q`, `residual`, the cache and the
tables as they are at the launch, so a serving loop writes the next token's into them and launches again, or replays a graph that captured
the launch.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import ClassVar

from intent_amd.examples.kernels.contraction import linear_i8
from intent_amd.examples.kernels.normalization import quantize_rows, residual_norm
from intent_amd.examples.kernels.streaming import prefix_decode
from intent_amd.runtime import PreparedSequence


@dataclass(frozen=True)
class Int8LayerStep:
    mutable_inputs: ClassVar[tuple[int, ...]] = ()     # no input is written
    attend: object           # JIT kernel of paged_gqa_decode_prefix
    narrow: object           # JIT kernel of quantize_rows
    product: object          # JIT kernel of linear_i8
    norm_narrow: object      # JIT kernel of residual_norm_i8
    gated_narrow: object     # JIT kernel of swiglu_quantize_rows
    norm: object             # JIT kernel of residual_norm

    @classmethod
    def from_jit(cls, jit, *, dtype, head_group):
        """Jit the kernels for rows of `dtype` ("f16" or "bf16") through `jit`."""
        return cls(attend=jit(getattr(prefix_decode, f"paged_gqa_decode_prefix_{dtype}"), constexprs=dict(HEAD_GROUP=head_group)),
                   narrow=jit(getattr(quantize_rows, f"quantize_rows_{dtype}")),
                   product=jit(getattr(linear_i8, f"linear_i8_{dtype}")),
                   norm_narrow=jit(getattr(residual_norm, f"residual_norm_i8_{dtype}")),
                   gated_narrow=jit(getattr(quantize_rows, f"swiglu_quantize_rows_{dtype}")),
                   norm=jit(getattr(residual_norm, f"residual_norm_{dtype}")))

    def prepare(self, q, key_cache, value_cache, prefix_indices, prefix_length, page_offsets, page_indices, sequence_lengths, scale,
                residual, out_weight, halves_weight, back_weight, block_norms, layer_norms, residual_scale, block_scale, eps, *,
                outputs=None):
        """`out_weight`, `halves_weight`, `back_weight`: the products'. `block_norms`, `layer_norms`: (post_weight, weight) of the norms
        behind the attention and behind the feed-forward block. `outputs`: the stream's and the next input's buffers."""
        scales = (residual_scale, block_scale, eps)
        ungated = block_norms[1].new_empty(0)
        attend = self.attend.prepare(q, key_cache, value_cache, prefix_indices, prefix_length, page_offsets, page_indices,
                                     sequence_lengths, scale)
        heads = self.narrow.prepare(attend.result().flatten(1))
        project = self._product(heads.result(), out_weight)
        middle = self.norm_narrow.prepare(project.result(), residual, ungated, *block_norms, *scales)
        stream, *rows = middle.result()
        halves = self._product(rows, halves_weight)
        gate, up = halves.result().chunk(2, 1)
        gated = self.gated_narrow.prepare(gate, up)
        back = self._product(gated.result(), back_weight)
        last = self.norm.prepare(back.result(), stream, ungated, *layer_norms, *scales, outputs=outputs)
        return PreparedSequence((attend, heads, project, middle, halves, gated, back, last), outputs=last.result())

    def _product(self, rows, weight):
        elements, row_scales = rows
        whole, scales, bias = weight
        return self.product.prepare(elements, whole, row_scales, scales, bias)

    def run(self, *arguments, **bindings):
        prepared = self.prepare(*arguments, **bindings)
        prepared.launch()
        return prepared.result()
