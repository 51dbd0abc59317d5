"""Definitions the hip provider recognises, and how each is launched.

A definition is recognised by its name plus its runtime signature (access kind,
dtype and rank of every parameter, constexpr names). The signature check stops a
same-named definition with a different contract from being routed to a kernel.
Recognised definitions (reference file:line of the semantics each kernel follows):

  stable_softmax          normalization/softmax.py:23-36   intent_hip_softmax_fwd (f32)
  stable_softmax_f16      normalization/softmax.py:39-51   intent_hip_softmax_fwd (f16)
  chunked_softmax_bf16    normalization/softmax.py:54-66   intent_hip_softmax_fwd (bf16)
  softmax_backward        backward/softmax.py:9-25         intent_hip_softmax_bwd (f32)
  softmax_backward_f16    f16-storage variant of the same  intent_hip_softmax_bwd (f16)
  gemm_f32                contraction/gemm.py:15-27        intent_hip_gemm_f32 (transpose_b 0)
  linear_f32              contraction/gemm.py:30-38        intent_hip_gemm_f32 (transpose_b 1)
  gemm_i8                 contraction/gemm.py:41-51        intent_hip_gemm_i8
  gemm                    contraction/gemm.py:54-73        intent_hip_gemm (f16, ACTIVATION)
  quantized_gemm          contraction/gemm.py:95-121       intent_hip_quantized_gemm
  bf16_gemm               contraction/gemm.py:76-92        intent_hip_gemm_bf16
  flash_attention_fwd     streaming/attention.py:428-466   intent_hip_attention_fwd_f16
  flash_gqa_attention_fwd streaming/attention.py:469-507   intent_hip_attention_fwd (f16, HEAD_GROUP)
  flash_attention_bf16_fwd streaming/attention.py:510-553  intent_hip_attention_fwd (bf16, HEAD_GROUP)
  flash_attention_bias_fwd streaming/attention.py:800-836  intent_hip_attention_bias_fwd
  mla_prefill             streaming/attention.py:756-798   intent_hip_mla_prefill (HEAD_GROUP, causal)
  flash_varlen_attention_fwd streaming/attention.py:839-877 intent_hip_attention_varlen_fwd (one head, CAUSAL)
  flash_varlen_gqa_prefill streaming/attention.py:880-924  intent_hip_attention_varlen_fwd (HEAD_GROUP, causal)
  csr_spmv                sparse/csr_spmv.py:11-29         intent_hip_csr_spmv_f32
  attention_backward_delta backward/attention.py:17-34     intent_hip_attention_bwd_delta
  attention_backward_dkdv backward/attention.py:87-137     intent_hip_attention_bwd_dkdv
  attention_backward_dq   backward/attention.py:171-211    intent_hip_attention_bwd_dq
  paged_gqa_decode_partials streaming/paged_attention.py:77-165  intent_hip_paged_decode_partials
  splitk_attention_f32_to_f16_reduce streaming/splitk_reduce.py:129-155  intent_hip_splitk_reduce_f32_to_f16
  grouped_flash_decode_partials streaming/attention.py:556-627  intent_hip_grouped_decode_partials
  continuous_gqa_decode   streaming/attention.py:629-670   intent_hip_continuous_gqa_decode
  varlen_gqa_decode_with_sink_logits streaming/attention.py:672-754  intent_hip_varlen_decode_sink
  csr_spmm                sparse/csr_spmm.py:11-33         intent_hip_csr_spmm_f32

(paths relative to python/intent/examples/kernels/ in the reference), and of this package alone:

  qk_norm_rope_{f16,bf16}           normalization/qk_norm_rope.py  intent_hip_qk_norm_rope
  qk_norm_rope_backward_{f16,bf16}  backward/qk_norm_rope.py       intent_hip_qk_norm_rope_backward
  paged_cache_append_{f16,bf16}     streaming/mx_cache.py          intent_hip_paged_cache_append
  paged_cache_read_{f16,bf16}       streaming/mx_cache.py          intent_hip_paged_cache_read
  paged_gqa_decode_mx_{f16,bf16}    streaming/mx_cache.py          intent_hip_paged_gqa_decode_mx
  linear_mxfp4_{f16,bf16}           contraction/linear_mxfp4.py    intent_hip_linear_mxfp4
  residual_norm_{f16,bf16}          normalization/residual_norm.py intent_hip_residual_norm
  residual_norm_i8_{f16,bf16}       normalization/residual_norm.py intent_hip_residual_norm_i8
  residual_norm_backward_{f16,bf16} backward/residual_norm.py      intent_hip_residual_norm_backward
  quantize_rows_{f16,bf16}          normalization/quantize_rows.py intent_hip_quantize_rows
  swiglu_quantize_rows_{f16,bf16}   normalization/quantize_rows.py intent_hip_swiglu_quantize_rows
  linear_i8_{f16,bf16}              contraction/linear_i8.py       intent_hip_linear_i8
  paged_gqa_decode_prefix_{f16,bf16} streaming/prefix_decode.py    intent_hip_paged_gqa_decode_prefix

Layout handling: kernels read rows with unit inner stride. An input whose inner
stride is not 1 is copied into a contiguous device buffer at every launch (on
the launch stream, so the copy sees the values current at launch time); an Out
buffer with a non-unit inner stride receives the result through a contiguous
buffer copied back after the kernel.
"""
from __future__ import annotations

import contextlib
import contextvars
import functools
from dataclasses import dataclass, field
from typing import Callable

from ...diagnostics import CompilationStageError
from ..torch_views import raw_stream_getter
from .library import (BF16, F16, F32, STATIC_SCRATCH_BYTES, OP_ATTENTION_BWD_DELTA, OP_ATTENTION_BWD_DKDV, OP_ATTENTION_BWD_DQ,
                      OP_ATTENTION_FWD, OP_ATTENTION_FWD_F16, OP_ATTENTION_BIAS, OP_ATTENTION_VARLEN, OP_MLA_PREFILL, OP_CSR_SPMV_F32, OP_GEMM, OP_GEMM_F32, OP_GEMM_I8, OP_QUANTIZED_GEMM,
                      OP_CSR_SPMM_F32, OP_CONTINUOUS_DECODE, OP_GROUPED_DECODE_PARTIALS, OP_PAGED_DECODE_PARTIALS, OP_PAGED_CACHE_APPEND, OP_PAGED_CACHE_READ, OP_PAGED_GQA_DECODE_MX, OP_LINEAR_MXFP4, OP_LINEAR_I8, OP_PAGED_GQA_DECODE_PREFIX, OP_QUANTIZE_ROWS, OP_SWIGLU_QUANTIZE_ROWS,
                      OP_RESIDUAL_NORM, OP_RESIDUAL_NORM_BACKWARD, OP_RESIDUAL_NORM_I8, OP_QK_NORM_ROPE, OP_QK_NORM_ROPE_BACKWARD, OP_VARLEN_DECODE, OP_SOFTMAX_BWD, OP_SOFTMAX_FWD, OP_SPLITK_REDUCE)


@dataclass
class Launch:
    """A bound native call: `run(stream)` returns the ABI status."""

    entry: str
    run: Callable[[int], int]
    keep: tuple = ()
    before: tuple = ()            # callables run on the launch stream before the kernel
    after: tuple = ()             # callables run on the launch stream after the kernel
    configuration: tuple = ()
    resources: Callable[[], dict | None] = field(default=lambda: None)
    candidates: tuple = ()        # (row, eligible, reasons) of the definition's tuning family, table order
    # The launch of other arguments of the same layout (shapes, strides, types, alignment to 16 bytes), in declaration order;
    # holds no tensor. None where a plan has to look at its arguments again.
    again: Callable[[tuple], "Launch"] | None = None


@dataclass(frozen=True)
class OperatorSpec:
    name: str
    signature: tuple              # per runtime parameter: ("view", access, dtype, rank) | ("scalar", dtype)
    constexprs: tuple[str, ...]
    plan: Callable
    # An Out may be exactly one of the inputs (same address and strides): True, or the pairs of positions of which that holds.
    inplace_safe: bool | frozenset = False
    derived: tuple = ()           # (symbol, source symbol, offset): extent(symbol) = extent(source) + offset
    repeats: bool = False         # its launches can be made again for other arguments of their layout (Launch.again)

    def may_be_one(self, left: int, right: int) -> bool:
        """Whether the parameters at two positions, of which one is written, may be the same view."""
        return self.inplace_safe is True or bool(self.inplace_safe) and (left, right) in self.inplace_safe

    @property
    def entry_point(self) -> str:
        """The C-ABI function (include/intent_hip.h) a launch of this definition calls."""
        return ENTRY_POINTS[self.name]


IN, OUT, INOUT = 0, 1, 2


def _view(access, dtype, rank):
    return ("view", access, dtype, rank)


# ------------------------------------------------------------------------------ workspace policy
# The target's backend_options["workspace"]: "prepare" lets a plan allocate device memory once per
# prepared call (staging copies, SpMV plan, split partial sums); "static" forbids it.
_WORKSPACE = contextvars.ContextVar("intent_hip_workspace", default="prepare")


@contextlib.contextmanager
def workspace_policy(policy: str):
    """Plans made inside this block follow `policy` ("prepare" or "static")."""
    token = _WORKSPACE.set(policy)
    try:
        yield
    finally:
        _WORKSPACE.reset(token)


def _static_workspace() -> bool:
    return _WORKSPACE.get() == "static"


# The program's compile options numerics: "source" keeps every low-precision cast where the
# definition puts it; "relaxed_normalization" lets a plan pick a kernel that applies the
# normalized-summary rewrite.
_NUMERICS = contextvars.ContextVar("intent_hip_numerics", default="source")


@contextlib.contextmanager
def numerics_policy(numerics: str):
    token = _NUMERICS.set(numerics)
    try:
        yield
    finally:
        _NUMERICS.reset(token)


def _relaxed_normalization() -> bool:
    return _NUMERICS.get() == "relaxed_normalization"


# The program's rows of its tuning family (runtime/hip/tuning.py), in table order.
_TUNING = contextvars.ContextVar("intent_hip_tuning", default=None)


@contextlib.contextmanager
def tuning_policy(rows):
    token = _TUNING.set(rows)
    try:
        yield
    finally:
        _TUNING.reset(token)


class plan_policies:
    """workspace_policy, numerics_policy and tuning_policy at once, for the plan of one call."""

    __slots__ = ("_values", "_tokens")

    def __init__(self, workspace: str, numerics: str, rows):
        self._values = (workspace, numerics, rows)

    def __enter__(self):
        workspace, numerics, rows = self._values
        self._tokens = (_WORKSPACE.set(workspace), _NUMERICS.set(numerics), _TUNING.set(rows))

    def __exit__(self, *_):
        workspace, numerics, rows = self._tokens
        _TUNING.reset(rows)
        _NUMERICS.reset(numerics)
        _WORKSPACE.reset(workspace)


def _split_choice(family: str, split_bytes: int) -> tuple[int, tuple]:
    """The first eligible row of `family` (columns: split) and every row's assessment. split = 1
    needs a grid small enough to split (split_bytes > 0: the workspace it takes) and a workspace
    policy that allows one; split = 0 is always eligible."""
    from .tuning import DEFAULT_FAMILIES

    rows = _TUNING.get() or DEFAULT_FAMILIES[family]
    candidates, chosen = [], None
    for row in rows:
        reasons = []
        if row[0] == 1:
            if _static_workspace():
                reasons.append("backend_options workspace='static' allows no workspace")
            if split_bytes <= 0:
                reasons.append("nothing to split: the grid fills the device or the walk is too short")
        candidates.append((row, not reasons, tuple(reasons)))
        if not reasons and chosen is None:
            chosen = row[0]
    if chosen is None:
        raise CompilationStageError("provider_configuration",
                                    f"no row of tuning family {family} is eligible for this call: "
                                    + "; ".join(f"{list(r)}: {', '.join(why)}" for r, _, why in candidates))
    return chosen, tuple(candidates)


# ------------------------------------------------------------------------------ layout helpers
def _aligned(tensor, vector: int) -> bool:
    """Unit inner stride, outer strides multiples of `vector` elements, 16-byte aligned start."""
    if tensor.numel() == 0 or tensor.dim() == 0:
        return True
    if tensor.stride(-1) != 1 and tensor.shape[-1] > 1:
        return False
    if vector > 1:
        if tensor.data_ptr() % 16:
            return False
        if any(s % vector for s, e in zip(tensor.stride()[:-1], tensor.shape[:-1]) if e > 1):
            return False
    return True


def _readable(tensor, keep, before, vector: int = 1):
    """A tensor with the contents of `tensor` at launch time whose layout the kernel takes
    (unit inner stride; with `vector`, also aligned for 16-byte loads)."""
    if _aligned(tensor, vector):
        return tensor
    _refuse_staging(tensor, vector)
    staged = tensor.new_empty(tensor.shape)
    keep.append(staged)
    before.append(lambda: staged.copy_(tensor))
    return staged


def _writable(tensor, keep, after, vector: int = 1):
    if _aligned(tensor, vector):
        return tensor
    _refuse_staging(tensor, vector)
    staged = tensor.new_empty(tensor.shape)
    keep.append(staged)
    after.append(lambda: tensor.copy_(staged))
    return staged


def _refuse_staging(tensor, vector: int) -> None:
    if _static_workspace():
        need = "unit inner stride" + (f", outer strides in multiples of {vector} and a 16-byte aligned start"
                                      if vector > 1 else "")
        raise ValueError(f"with backend_options workspace='static' the provider does not stage views; this "
                         f"kernel needs {need}, got strides {tuple(tensor.stride())}")


def _workspace_run(fn, args, size, device, keep):
    """The launch fn(*args, workspace, size, stream) with a workspace allocated here. That one is ordered with the stream it
    was allocated on and may be freed with the call, so a launch on another stream, or into a graph (never on stream 0),
    takes one that belongs to that stream or graph."""
    import torch

    home = raw_stream_getter()(device.index)
    kept = torch.empty(size, dtype=torch.uint8, device=device)
    keep.append(kept)
    address, capturing = kept.data_ptr(), torch.cuda.is_current_stream_capturing

    def run(stream):
        if stream == home and (stream == 0 or not capturing()):
            return fn(*args, address, size, stream)
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        return fn(*args, workspace.data_ptr(), size, stream)
    return run


def _optional_workspace_run(fn, args, size, device, keep):
    return _workspace_run(fn, args, size, device, keep) if size else lambda stream: fn(*args, None, 0, stream)


def _staged(again, values, bound, before, after):
    """The launch of `values`, which hold staged views where `before` and `after` copy them: such a launch is planned anew for
    other arguments."""
    launch = again(values)
    if before or after:
        launch.keep, launch.before, launch.after = (*launch.keep, bound.arguments), tuple(before), tuple(after)
    else:
        launch.again = again
    return launch


# ------------------------------------------------------------------------------ attention head dimensions
# The attention kernels are built for key and value head dimensions of 64 and 128. Any other width up
# to 128 (the reference declares D and DV symbolic, streaming/attention.py:428-553) runs on the next of
# the two through zero-padded copies refreshed at each launch: zero dimensions add exact zeros to
# every score's sum and give output columns that are dropped, so results equal the unpadded ones.
_KERNEL_WIDTHS = (64, 128)


def _kernel_width(extent: int, name: str) -> int:
    for width in _KERNEL_WIDTHS:
        if extent <= width:
            return width
    raise CompilationStageError("provider_configuration",
                                f"{name} = {extent}: the hip attention kernels take head dimensions up to "
                                f"{_KERNEL_WIDTHS[-1]}")


def _padded_in(tensor, width, keep, before):
    """`tensor` with its last dimension extended to `width` by zeros; the copy runs at each launch."""
    _refuse_staging(tensor, 8)
    staged = tensor.new_zeros(tuple(tensor.shape[:-1]) + (width,))
    head = staged[..., :tensor.shape[-1]]
    keep.append(staged)
    before.append(lambda: head.copy_(tensor))
    return staged


def _padded_out(tensor, width, keep, after):
    """A buffer of last dimension `width` whose first columns are copied into `tensor` after a launch."""
    _refuse_staging(tensor, 8)
    staged = tensor.new_empty(tuple(tensor.shape[:-1]) + (width,))
    head = staged[..., :tensor.shape[-1]]
    keep.append(staged)
    after.append(lambda: tensor.copy_(head))
    return staged


def _attention_views(q, k, v, o, keep, before, after):
    """q, k, v and o as an attention kernel reads them, and the kernel's (d, dv): unit inner stride,
    16-byte aligned rows, head dimensions padded to 64 or 128 where they are not."""
    d, dv = q.shape[-1], v.shape[-1]
    kd, kdv = _kernel_width(d, "d"), _kernel_width(dv, "dv")
    if kd != d:
        qk, kk = _padded_in(q, kd, keep, before), _padded_in(k, kd, keep, before)
    else:
        qk, kk = _readable(q, keep, before, 8), _readable(k, keep, before, 8)
    if kdv != dv:
        vk, ok = _padded_in(v, kdv, keep, before), _padded_out(o, kdv, keep, after)
    else:
        vk, ok = _readable(v, keep, before, 8), _writable(o, keep, after, 8)
    return qk, kk, vk, ok, kd, kdv


def _row_stride(tensor):
    rows, cols = tensor.shape
    return tensor.stride(0) if rows > 1 else cols


# ------------------------------------------------------------------------------ softmax
def _softmax_fwd(dtype_code):
    def plan(lib, bound, constexprs, device):
        x, y = bound.arguments
        keep, before, after = [x, y], [], []
        xk, yk = _readable(x, keep, before), _writable(y, keep, after)
        rows, cols = x.shape
        fn = lib.fn["softmax_fwd"]
        args = (dtype_code, xk.data_ptr(), yk.data_ptr(), rows, cols, _row_stride(xk), _row_stride(yk))
        return Launch("intent_hip_softmax_fwd", lambda stream: fn(*args, stream), tuple(keep), tuple(before),
                      tuple(after), (("rows", rows), ("cols", cols)),
                      lambda: lib.call_resources(OP_SOFTMAX_FWD, *args))
    return plan


def _softmax_bwd(dtype_code):
    def plan(lib, bound, constexprs, device):
        p, dy, dx = bound.arguments
        keep, before, after = [p, dy, dx], [], []
        pk, gk, dk = _readable(p, keep, before), _readable(dy, keep, before), _writable(dx, keep, after)
        rows, cols = p.shape
        fn = lib.fn["softmax_bwd"]
        args = (dtype_code, pk.data_ptr(), gk.data_ptr(), dk.data_ptr(), rows, cols, _row_stride(pk),
                _row_stride(gk), _row_stride(dk))
        return Launch("intent_hip_softmax_bwd", lambda stream: fn(*args, stream), tuple(keep), tuple(before),
                      tuple(after), (("rows", rows), ("cols", cols)),
                      lambda: lib.call_resources(OP_SOFTMAX_BWD, *args))
    return plan


# ------------------------------------------------------------------------------ GEMM
def _split_bytes(lib, name, m, n, k) -> int:
    """Bytes of the f32 sums of a product whose K is divided over workgroups; 0 where nothing is split (enough output
    tiles, or workspace='static')."""
    import ctypes

    size = ctypes.c_size_t(0)
    lib.check(lib.fn[name + "_workspace_bytes"](m, n, k, ctypes.byref(size)), "provider_preparation")
    return 0 if _static_workspace() else size.value


def _gemm_launch(lib, dtype_code, activation, a, b, c, entry, configuration, device):
    keep, before, after = [a, b, c], [], []
    ak, bk, ck = _readable(a, keep, before), _readable(b, keep, before), _writable(c, keep, after)
    m, k = a.shape
    n = b.shape[1]
    args = product = (ak.data_ptr(), bk.data_ptr(), ck.data_ptr(), m, n, k, _row_stride(ak), _row_stride(bk), _row_stride(ck))
    facts = (("m", m), ("n", n), ("k", k)) + configuration
    resources = lambda: lib.call_resources(OP_GEMM, dtype_code, *product, activation)  # noqa: E731
    size = _split_bytes(lib, "gemm", m, n, k)
    if size:
        entry, facts = "intent_hip_gemm_ws", facts + (("workspace_bytes", size),)
        run = _workspace_run(lib.fn["gemm_ws"], (dtype_code, activation, *args), size, device, keep)
    else:
        if entry == "intent_hip_gemm_bf16":
            fn = lib.fn["gemm_bf16"]
        else:
            fn, args = lib.fn["gemm"], (dtype_code, activation, *args)
        run = lambda stream: fn(*args, stream)  # noqa: E731
    return Launch(entry, run, tuple(keep), tuple(before), tuple(after), facts, resources)


def _gemm_bf16(lib, bound, constexprs, device):
    return _gemm_launch(lib, BF16, 0, *bound.arguments, "intent_hip_gemm_bf16", (), device)


def _activation_code(value) -> int:
    """ACTIVATION constexpr (an Activation enum member, gemm.py:10-12) -> ABI code."""
    code = getattr(value, "value", value)
    if code not in (0, 1):
        raise CompilationStageError("provider_configuration",
                                    f"the hip gemm supports ACTIVATION NONE (0) or RELU (1), got {value!r}")
    return int(code)


def _gemm16(dtype_code):
    def plan(lib, bound, constexprs, device):
        activation = _activation_code(constexprs.get("ACTIVATION", 0))
        return _gemm_launch(lib, dtype_code, activation, *bound.arguments, "intent_hip_gemm",
                            (("activation", activation),), device)
    return plan


def _gemm_f32(transpose_b: bool):
    def plan(lib, bound, constexprs, device):
        a, b, c = bound.arguments
        keep, before, after = [a, b, c], [], []
        ak, bk, ck = _readable(a, keep, before), _readable(b, keep, before), _writable(c, keep, after)
        m, k = a.shape
        n = b.shape[0] if transpose_b else b.shape[1]
        args = (ak.data_ptr(), bk.data_ptr(), ck.data_ptr(), m, n, k, _row_stride(ak), _row_stride(bk),
                _row_stride(ck), int(transpose_b))
        facts = (("m", m), ("n", n), ("k", k), ("transpose_b", transpose_b))
        fn, entry = lib.fn["gemm_f32"], "intent_hip_gemm_f32"
        run = lambda stream: fn(*args, stream)  # noqa: E731
        size = _split_bytes(lib, "gemm_f32", m, n, k)
        if size:
            entry, facts = "intent_hip_gemm_f32_ws", facts + (("workspace_bytes", size),)
            run = _workspace_run(lib.fn["gemm_f32_ws"], args, size, device, keep)
        return Launch(entry, run, tuple(keep), tuple(before), tuple(after), facts,
                      lambda: lib.call_resources(OP_GEMM_F32, F32, *args))
    return plan


def _gemm_i8(lib, bound, constexprs, device):
    a, b, bias, c = bound.arguments
    keep, before, after = [a, b, bias, c], [], []
    ak, bk, biask, ck = (_readable(a, keep, before), _readable(b, keep, before), _readable(bias, keep, before),
                         _writable(c, keep, after))
    m, k = a.shape
    n = b.shape[1]
    fn = lib.fn["gemm_i8"]
    args = (ak.data_ptr(), bk.data_ptr(), biask.data_ptr(), ck.data_ptr(), m, n, k, _row_stride(ak), _row_stride(bk),
            _row_stride(ck))
    return Launch("intent_hip_gemm_i8", lambda stream: fn(*args, stream), tuple(keep), tuple(before), tuple(after),
                  (("m", m), ("n", n), ("k", k)), lambda: lib.kernel_resources(OP_GEMM_I8, 0, m, n))


def _quantized_gemm(lib, bound, constexprs, device):
    a, b, bias, residual, scale, out = bound.arguments
    keep, before, after = [a, b, bias, residual, scale, out], [], []
    ak, bk = _readable(a, keep, before), _readable(b, keep, before)
    biask, rk, sk = _readable(bias, keep, before), _readable(residual, keep, before), _readable(scale, keep, before)
    ok = _writable(out, keep, after)
    m, k = a.shape
    n = b.shape[1]
    fn = lib.fn["quantized_gemm"]
    args = (ak.data_ptr(), bk.data_ptr(), biask.data_ptr(), rk.data_ptr(), sk.data_ptr(), ok.data_ptr(), m, n, k,
            _row_stride(ak), _row_stride(bk), _row_stride(rk), _row_stride(ok))
    return Launch("intent_hip_quantized_gemm", lambda stream: fn(*args, stream), tuple(keep), tuple(before),
                  tuple(after), (("m", m), ("n", n), ("k", k)),
                  lambda: lib.call_resources(OP_QUANTIZED_GEMM, F16, args[0], args[1], args[3], *args[5:]))


# ------------------------------------------------------------------------------ attention
def _attention_launch(lib, dtype_code, q, k, v, o, scale, group, causal, entry, device):
    """The batched attention forward (head_group query heads per key head). A grid too small to fill
    the device splits each query block's keys over workgroups through a workspace (tuning family
    hip.attention_forward; with workspace='static' or the unsplit row the launch stays unsplit)."""
    import ctypes

    import torch

    keep, before, after = [q, k, v, o], [], []
    qk, kk, vk, ok, d, dv = _attention_views(q, k, v, o, keep, before, after)
    batch, q_heads, sq = q.shape[:3]
    sk = k.shape[2]
    strides = (ctypes.c_int64 * 16)(*(s for t in (qk, kk, vk, ok) for s in t.stride()))
    keep.append(strides)
    size = ctypes.c_size_t(0)
    lib.check(lib.fn["attention_fwd_workspace_bytes"](batch, q_heads, sq, sk, dv, ctypes.byref(size)),
              "provider_preparation")
    split, candidates = _split_choice("hip.attention_forward", size.value)
    config = (("batch", batch), ("q_heads", q_heads), ("head_group", group), ("sq", sq), ("sk", sk), ("d", d),
              ("dv", dv), ("causal", causal), ("split", split))
    resources = lambda: lib.kernel_resources(OP_ATTENTION_FWD, dtype_code, sq, d | (dv << 16))  # noqa: E731
    if split:
        workspace = torch.empty(size.value, dtype=torch.uint8, device=device)
        keep.append(workspace)
        fn = lib.fn["attention_fwd_ws"]
        args = (dtype_code, qk.data_ptr(), kk.data_ptr(), vk.data_ptr(), ok.data_ptr(), batch, q_heads, group, sq,
                sk, d, dv, strides, float(scale), int(causal), workspace.data_ptr(), size.value)
        return Launch("intent_hip_attention_fwd_ws", lambda stream: fn(*args, stream), tuple(keep), tuple(before),
                      tuple(after), config, resources, candidates)
    if entry == "intent_hip_attention_fwd_f16":
        fn = lib.fn["attention_fwd_f16"]
        args = (qk.data_ptr(), kk.data_ptr(), vk.data_ptr(), ok.data_ptr(), batch, q_heads, sq, sk, d, dv, strides,
                float(scale), int(causal))
    else:
        fn = lib.fn["attention_fwd"]
        args = (dtype_code, qk.data_ptr(), kk.data_ptr(), vk.data_ptr(), ok.data_ptr(), batch, q_heads, group, sq,
                sk, d, dv, strides, float(scale), int(causal))
    return Launch(entry, lambda stream: fn(*args, stream), tuple(keep), tuple(before), tuple(after), config,
                  resources if entry != "intent_hip_attention_fwd_f16"
                  else (lambda: lib.kernel_resources(OP_ATTENTION_FWD_F16, F16, sq, d | (dv << 16))), candidates)


def _attention_f16(lib, bound, constexprs, device):
    q, k, v, o, scale = bound.arguments
    return _attention_launch(lib, F16, q, k, v, o, scale, 1, bool(constexprs["CAUSAL"]),
                             "intent_hip_attention_fwd_f16", device)


def _attention_grouped(dtype_code):
    """flash_gqa_attention_fwd (f16) / flash_attention_bf16_fwd (bf16): key head = query head //
    HEAD_GROUP (attention.py:485, 528)."""
    def plan(lib, bound, constexprs, device):
        q, k, v, o, scale = bound.arguments
        group = constexprs["HEAD_GROUP"]
        if isinstance(group, bool) or not isinstance(group, int) or group < 1:
            raise CompilationStageError("provider_configuration", f"HEAD_GROUP must be a positive int, got {group!r}")
        if k.shape[1] * group != q.shape[1]:
            raise ValueError(f"query heads ({q.shape[1]}) must equal key/value heads ({k.shape[1]}) * HEAD_GROUP "
                             f"({group})")
        return _attention_launch(lib, dtype_code, q, k, v, o, scale, group, bool(constexprs["CAUSAL"]),
                                 "intent_hip_attention_fwd", device)
    return plan


def _attention_bias(lib, bound, constexprs, device):
    """flash_attention_bias_fwd: scores (q . k) scale + bias[b, h, key] over every key, no mask
    (attention.py:800-836, :328-366)."""
    import ctypes

    q, k, v, bias, o, scale = bound.arguments
    batch, heads, sq = q.shape[:3]
    sk = k.shape[2]
    if tuple(bias.shape) != (batch, heads, sk):
        raise ValueError(f"bias must be [B, H, K] = {(batch, heads, sk)}, got {tuple(bias.shape)}")
    keep, before, after = [q, k, v, bias, o], [], []
    qk, kk, vk, ok, d, dv = _attention_views(q, k, v, o, keep, before, after)
    bk = _readable(bias, keep, before)
    strides = (ctypes.c_int64 * 16)(*(s for t in (qk, kk, vk, ok) for s in t.stride()))
    bias_strides = (ctypes.c_int64 * 3)(*bk.stride())
    keep += [strides, bias_strides]
    fn = lib.fn["attention_bias_fwd"]
    args = (qk.data_ptr(), kk.data_ptr(), vk.data_ptr(), bk.data_ptr(), ok.data_ptr(), batch, heads, sq, sk, d, dv,
            strides, bias_strides, float(scale))
    return Launch("intent_hip_attention_bias_fwd", lambda stream: fn(*args, stream), tuple(keep), tuple(before),
                  tuple(after), (("batch", batch), ("heads", heads), ("sq", sq), ("sk", sk), ("d", d), ("dv", dv)),
                  lambda: lib.kernel_resources(OP_ATTENTION_BIAS, F16, sq, d | (dv << 16)))


def _mla_prefill(lib, bound, constexprs, device):
    """mla_prefill: causal latent attention, scores (q . k + qpe . kpe) scale (attention.py:756-798)."""
    import ctypes

    import torch

    q, qpe, k, kpe, v, o, scale = bound.arguments
    group = _head_group(constexprs)
    batch, heads, sq, d = q.shape
    sk, p = k.shape[2], qpe.shape[3]
    if k.shape[1] * group != heads or v.shape[1] != k.shape[1]:
        raise ValueError(f"query heads ({heads}) must equal key/value heads ({k.shape[1]}) * HEAD_GROUP ({group})")
    keep, before, after = [q, qpe, k, kpe, v, o], [], []
    views = [_readable(t, keep, before, 8) for t in (q, qpe, k, kpe, v)] + [_writable(o, keep, after, 8)]
    strides = _strides(*views)
    keep.append(strides)
    # Small grids split the keys over workgroups through a workspace (tuning family
    # hip.latent_prefill; with workspace='static' or the unsplit row the launch stays unsplit).
    size = ctypes.c_size_t(0)
    lib.check(lib.fn["mla_prefill_workspace_bytes"](batch, heads, sq, sk, d, ctypes.byref(size)), "provider_preparation")
    split, candidates = _split_choice("hip.latent_prefill", size.value)
    workspace = None
    if split:
        workspace = torch.empty(size.value, dtype=torch.uint8, device=device)
        keep.append(workspace)
    fn = lib.fn["mla_prefill"]
    args = (*(t.data_ptr() for t in views), batch, heads, group, sq, sk, d, p, strides, float(scale),
            workspace.data_ptr() if workspace is not None else None, size.value if workspace is not None else 0)
    return Launch("intent_hip_mla_prefill", lambda stream: fn(*args, stream), tuple(keep), tuple(before),
                  tuple(after), (("batch", batch), ("heads", heads), ("head_group", group), ("sq", sq), ("sk", sk),
                                 ("d", d), ("p", p), ("split", split)),
                  lambda: lib.kernel_resources(OP_MLA_PREFILL, F16, sq, d | (p << 16)), candidates)


def _head_group(constexprs) -> int:
    group = constexprs["HEAD_GROUP"]
    if isinstance(group, bool) or not isinstance(group, int) or group < 1:
        raise CompilationStageError("provider_configuration", f"HEAD_GROUP must be a positive int, got {group!r}")
    return group


def _attention_varlen(grouped: bool):
    """flash_varlen_attention_fwd (q [U,D], one head, CAUSAL) / flash_varlen_gqa_prefill (q [U,HQ,D],
    key head = query head // HEAD_GROUP, causal): packed sequences delimited by cu_seqlens
    (attention.py:839-924). The offsets stay on the device: the kernel's own pre-pass lists the
    work items into a workspace allocated here, once per prepared call."""
    def plan(lib, bound, constexprs, device):
        import ctypes

        import torch

        q, k, v, lengths, cu, o, scale = bound.arguments
        if grouped:
            group, causal = _head_group(constexprs), True
            total, q_heads, d = q.shape
            if k.shape[1] * group != q_heads or v.shape[1] != k.shape[1]:
                raise ValueError(f"query heads ({q_heads}) must equal key/value heads ({k.shape[1]}) * HEAD_GROUP "
                                 f"({group})")
            dv = v.shape[2]
        else:
            group, causal = 1, bool(constexprs["CAUSAL"])
            (total, d), q_heads, dv = q.shape, 1, v.shape[1]
        sequences = lengths.shape[0]
        if cu.shape[0] != sequences + 1:
            raise ValueError(f"cu_seqlens needs sequence_lengths.shape[0] + 1 = {sequences + 1} entries, "
                             f"got {cu.shape[0]}")
        if k.shape[0] != total or v.shape[0] != total:
            raise ValueError("q, k and v must hold the same packed rows")
        if _static_workspace():
            raise CompilationStageError(
                "provider_preparation", "packed-sequence attention lists its work items in a workspace; "
                "backend_options workspace='static' has none for it, use workspace='prepare'")
        keep, before, after = [q, k, v, lengths, cu, o], [], []
        qk, kk, vk, ok, d, dv = _attention_views(q, k, v, o, keep, before, after)
        cuk = _readable(cu, keep, before)

        def row_head_inner(t):
            return (t.stride(0), t.stride(1), t.stride(2)) if t.dim() == 3 else (t.stride(0), 0, t.stride(1))

        strides = (ctypes.c_int64 * 12)(*(x for t in (qk, kk, vk, ok) for x in row_head_inner(t)))
        size = ctypes.c_size_t(0)
        lib.check(lib.fn["attention_varlen_workspace_bytes"](sequences, total, ctypes.byref(size)),
                  "provider_preparation")
        workspace = torch.empty(max(size.value, 1), dtype=torch.uint8, device=device)
        keep += [strides, workspace]
        fn = lib.fn["attention_varlen_fwd"]
        args = (F16, qk.data_ptr(), kk.data_ptr(), vk.data_ptr(), cuk.data_ptr(), ok.data_ptr(), sequences, total,
                q_heads, group, d, dv, strides, float(scale), int(causal), workspace.data_ptr(), size.value)
        return Launch("intent_hip_attention_varlen_fwd", lambda stream: fn(*args, stream), tuple(keep),
                      tuple(before), tuple(after),
                      (("sequences", sequences), ("total", total), ("q_heads", q_heads), ("head_group", group),
                       ("d", d), ("dv", dv), ("causal", causal), ("workspace_bytes", size.value)),
                      lambda: lib.kernel_resources(OP_ATTENTION_VARLEN, F16, total, d | (dv << 16)))
    return plan


# ------------------------------------------------------------------------------ attention backward
def _strides(*tensors):
    import ctypes

    values = [st for t in tensors for st in t.stride()]
    return (ctypes.c_int64 * len(values))(*values)


def _attention_bwd_delta(lib, bound, constexprs, device):
    o, dout, delta = bound.arguments
    keep, before, after = [o, dout, delta], [], []
    ok, gk = _readable(o, keep, before, 8), _readable(dout, keep, before, 8)
    batch, heads, sq, d = o.shape
    strides = _strides(ok, gk, delta)
    keep.append(strides)
    fn = lib.fn["attention_bwd_delta"]
    args = (ok.data_ptr(), gk.data_ptr(), delta.data_ptr(), batch, heads, sq, d, strides)
    return Launch("intent_hip_attention_bwd_delta", lambda stream: fn(*args, stream), tuple(keep), tuple(before),
                  tuple(after), (("batch", batch), ("heads", heads), ("sq", sq), ("d", d)),
                  lambda: lib.kernel_resources(OP_ATTENTION_BWD_DELTA, F16, sq, d))


def _backward_group(q, k, constexprs):
    group = constexprs["HEAD_GROUP"]
    if isinstance(group, bool) or not isinstance(group, int) or group < 1:
        raise CompilationStageError("provider_configuration", f"HEAD_GROUP must be a positive int, got {group!r}")
    if k.shape[1] * group != q.shape[1]:
        raise ValueError(f"query heads ({q.shape[1]}) must equal key/value heads ({k.shape[1]}) * HEAD_GROUP "
                         f"({group})")
    return group


def _attention_bwd(kind):
    """attention_backward_dq (kind "dq") / attention_backward_dkdv (kind "dkdv"); lse and delta are
    read through their own strides, 4-D operands with unit inner stride (staged otherwise)."""
    def plan(lib, bound, constexprs, device):
        if kind == "dq":
            q, k, v, dout, lse, delta, out, scale = bound.arguments
            outs = (out,)
        else:
            q, k, v, dout, lse, delta, grad_k, grad_v, scale = bound.arguments
            outs = (grad_k, grad_v)
        group = _backward_group(q, k, constexprs)
        causal = bool(constexprs["CAUSAL"])
        keep, before, after = [q, k, v, dout, lse, delta, *outs], [], []
        ins = [_readable(t, keep, before, 8) for t in (q, k, v, dout)]
        staged_outs = [_writable(t, keep, after, 8) for t in outs]
        batch, q_heads, sq, d = q.shape
        sk = k.shape[2]
        strides = _strides(*ins, lse, delta, *staged_outs)
        keep.append(strides)
        args = (*(t.data_ptr() for t in ins), lse.data_ptr(), delta.data_ptr(),
                *(t.data_ptr() for t in staged_outs), batch, q_heads, group, sq, sk, d, strides, float(scale),
                int(causal))
        configuration = (("batch", batch), ("q_heads", q_heads), ("head_group", group), ("sq", sq), ("sk", sk),
                         ("d", d), ("causal", causal))
        # Small grids split their work over more workgroups; the f32 partial sums need a
        # workspace, allocated here once per prepared call.
        import ctypes

        # (tuning family hip.attention_backward: split = 0 runs the unsplit kernels)
        size = ctypes.c_size_t(0)
        extents = (batch, q_heads, group, sq, sk, d)
        if kind == "dq":
            status = lib.fn["attention_bwd_dq_workspace_bytes"](*extents, ctypes.byref(size))
        else:
            status = lib.fn["attention_bwd_dkdv_masked_workspace_bytes"](*extents, int(causal), ctypes.byref(size))
        lib.check(status, "provider_preparation")
        split, candidates = _split_choice("hip.attention_backward", size.value)
        fn = lib.fn[f"attention_bwd_{kind}_ws"]
        if split:
            run = _workspace_run(fn, args, size.value, device, keep)
        else:
            run = lambda stream: fn(*args, None, 0, stream)  # noqa: E731
        configuration += (("split", split), ("workspace_bytes", size.value if split else 0))
        if kind == "dq":   # the kernel variant depends on the rows of the call
            resources = lambda: lib.kernel_resources(OP_ATTENTION_BWD_DQ, F16, batch * q_heads * sq, d)  # noqa: E731
        else:
            resources = lambda: lib.call_resources(OP_ATTENTION_BWD_DKDV, F16, *extents, int(causal), split)  # noqa: E731
        return Launch(f"intent_hip_attention_bwd_{kind}", run, tuple(keep), tuple(before), tuple(after), configuration,
                      resources, candidates)
    return plan


# ------------------------------------------------------------------------------ paged decode
def _positive_constexpr(constexprs, name):
    value = constexprs[name]
    if isinstance(value, bool) or not isinstance(value, int) or value < 1:
        raise CompilationStageError("provider_configuration", f"{name} must be a positive int, got {value!r}")
    return value


def _paged_decode_partials(lib, bound, constexprs, device):
    """paged_gqa_decode_partials: one workgroup per (job, key head). The page tables are read as
    given; positions and physical pages outside their arrays are clamped by the kernel."""
    (q, key_cache, value_cache, page_offsets, page_indices, lengths, split_offsets, partial_lse, partial_output,
     scale) = bound.arguments
    page_size = _positive_constexpr(constexprs, "PAGE_SIZE")
    group = _positive_constexpr(constexprs, "HEAD_GROUP")
    splits = _positive_constexpr(constexprs, "SPLITS")
    batch, q_heads, d = q.shape
    pages, ps, kv_heads, dv = value_cache.shape
    if page_offsets.shape[0] != batch + 1:
        raise ValueError(f"page_offsets must hold batch + 1 = {batch + 1} entries, got {page_offsets.shape[0]}")
    if split_offsets.shape[0] != batch * splits + 1:
        raise ValueError(f"split_offsets must hold batch * SPLITS + 1 = {batch * splits + 1} entries, "
                         f"got {split_offsets.shape[0]}")
    if kv_heads * group != q_heads:
        raise ValueError(f"query heads ({q_heads}) must equal key/value heads ({kv_heads}) * HEAD_GROUP ({group})")
    keep = [q, key_cache, value_cache, page_offsets, page_indices, lengths, split_offsets, partial_lse,
            partial_output]
    before, after = [], []
    qk = _readable(q, keep, before)
    kk, vk = _readable(key_cache, keep, before, 8), _readable(value_cache, keep, before, 8)
    tables = [_readable(t, keep, before) for t in (page_offsets, page_indices, lengths, split_offsets)]
    ok = _writable(partial_output, keep, after)
    strides = _strides(qk, kk, vk, partial_lse, ok)
    keep.append(strides)
    fn = lib.fn["paged_decode_partials"]
    args = (qk.data_ptr(), kk.data_ptr(), vk.data_ptr(), *(t.data_ptr() for t in tables), partial_lse.data_ptr(),
            ok.data_ptr(), batch, q_heads, d, pages, ps, kv_heads, dv, page_indices.shape[0], page_size, group,
            splits, strides, float(scale))
    return Launch("intent_hip_paged_decode_partials", lambda stream: fn(*args, stream), tuple(keep), tuple(before),
                  tuple(after),
                  (("batch", batch), ("q_heads", q_heads), ("kv_heads", kv_heads), ("head_group", group),
                   ("d", d), ("pages", pages), ("ps", ps), ("page_size", page_size), ("splits", splits)),
                  lambda: lib.call_resources(OP_PAGED_DECODE_PARTIALS, F16, batch, kv_heads, group, d,
                                             page_indices.shape[0], ps, splits))


def _grouped_decode_partials(lib, bound, constexprs, device):
    """grouped_flash_decode_partials: one workgroup per (batch, part, key head) over the bf16 caches."""
    q, k, v, partial_lse, partial_output, scale = bound.arguments
    group = _positive_constexpr(constexprs, "HEAD_GROUP")
    parts = _positive_constexpr(constexprs, "P")
    split = _positive_constexpr(constexprs, "SPLIT_SIZE")
    batch, q_heads, _, d = q.shape
    kv_heads, keys, dv = k.shape[1], k.shape[2], v.shape[3]
    if partial_lse.shape[2] != parts:
        raise ValueError(f"partial_lse holds {partial_lse.shape[2]} parts, P is {parts}")
    if kv_heads * group != q_heads:
        raise ValueError(f"query heads ({q_heads}) must equal key/value heads ({kv_heads}) * HEAD_GROUP ({group})")
    keep, before, after = [q, k, v, partial_lse, partial_output], [], []
    qk, kk, vk = _readable(q, keep, before), _readable(k, keep, before, 8), _readable(v, keep, before, 8)
    lk, ok = _writable(partial_lse, keep, after), _writable(partial_output, keep, after)
    strides = _strides(qk, kk, vk, lk, ok)
    keep.append(strides)
    fn = lib.fn["grouped_decode_partials"]
    args = (qk.data_ptr(), kk.data_ptr(), vk.data_ptr(), lk.data_ptr(), ok.data_ptr(), batch, q_heads, kv_heads, group,
            keys, d, dv, parts, split, strides, float(scale))
    return Launch("intent_hip_grouped_decode_partials", lambda stream: fn(*args, stream), tuple(keep), tuple(before),
                  tuple(after), (("batch", batch), ("q_heads", q_heads), ("kv_heads", kv_heads), ("keys", keys),
                                 ("d", d), ("parts", parts), ("split_size", split)),
                  lambda: lib.kernel_resources(OP_GROUPED_DECODE_PARTIALS, BF16, group, d))


def _decode_workspace(name):
    if _static_workspace():
        raise CompilationStageError(
            "provider_preparation", f"{name} merges split states through a workspace; backend_options "
            "workspace='static' has none for it, use workspace='prepare'")


def _continuous_decode(lib, bound, constexprs, device):
    """continuous_gqa_decode: the keys split over (batch, split, key head) workgroups whose states
    merge in a second kernel, through a workspace allocated here."""
    import ctypes

    import torch

    q, k, v, mask, output, scale = bound.arguments
    group = _positive_constexpr(constexprs, "HEAD_GROUP")
    batch, q_heads, d = q.shape
    keys, kv_heads, dv = k.shape[1], k.shape[2], v.shape[3]
    if kv_heads * group != q_heads:
        raise ValueError(f"query heads ({q_heads}) must equal key/value heads ({kv_heads}) * HEAD_GROUP ({group})")
    _decode_workspace("continuous_gqa_decode")
    keep, before, after = [q, k, v, mask, output], [], []
    qk, kk, vk = _readable(q, keep, before), _readable(k, keep, before, 8), _readable(v, keep, before, 8)
    mk, ok = _readable(mask, keep, before), _writable(output, keep, after)
    strides = _strides(qk, kk, vk, mk, ok)
    size = ctypes.c_size_t(0)
    lib.check(lib.fn["dense_decode_workspace_bytes"](batch, q_heads, kv_heads, keys, dv, ctypes.byref(size)),
              "provider_preparation")
    workspace = torch.empty(max(size.value, 1), dtype=torch.uint8, device=device)
    keep += [strides, workspace]
    fn = lib.fn["continuous_gqa_decode"]
    args = (qk.data_ptr(), kk.data_ptr(), vk.data_ptr(), mk.data_ptr(), ok.data_ptr(), batch, q_heads, kv_heads, group,
            keys, d, dv, strides, float(scale), workspace.data_ptr(), size.value)
    return Launch("intent_hip_continuous_gqa_decode", lambda stream: fn(*args, stream), tuple(keep), tuple(before),
                  tuple(after), (("batch", batch), ("q_heads", q_heads), ("kv_heads", kv_heads), ("keys", keys),
                                 ("d", d), ("workspace_bytes", size.value)),
                  lambda: lib.kernel_resources(OP_CONTINUOUS_DECODE, F16, group, d))


def _varlen_decode(lib, bound, constexprs, device):
    """varlen_gqa_decode_with_sink_logits: packed sequences split over (sequence, split, key head)
    workgroups; the merge adds the sink and turns the block maxima (kept in block_logits) into
    block logits. The offsets stay on the device."""
    import ctypes

    import torch

    q, k, v, cu, sink, output, block_logits, scale = bound.arguments
    group = _positive_constexpr(constexprs, "HEAD_GROUP")
    max_blocks = _positive_constexpr(constexprs, "MAX_BLOCKS")
    sequences, q_heads, d = q.shape
    rows, kv_heads, dv = k.shape[0], k.shape[1], v.shape[2]
    if kv_heads * group != q_heads:
        raise ValueError(f"query heads ({q_heads}) must equal key/value heads ({kv_heads}) * HEAD_GROUP ({group})")
    if cu.shape[0] != sequences + 1:
        raise ValueError(f"cu_seqlens needs q.shape[0] + 1 = {sequences + 1} entries, got {cu.shape[0]}")
    if max_blocks > block_logits.shape[2]:
        raise ValueError(f"MAX_BLOCKS ({max_blocks}) exceeds the {block_logits.shape[2]} block_logits columns")
    _decode_workspace("varlen_gqa_decode_with_sink_logits")
    keep, before, after = [q, k, v, cu, sink, output, block_logits], [], []
    qk, kk, vk = _readable(q, keep, before), _readable(k, keep, before, 8), _readable(v, keep, before, 8)
    cuk, sk = _readable(cu, keep, before), _readable(sink, keep, before)
    ok, bk = _writable(output, keep, after), _writable(block_logits, keep, after)
    strides = _strides(qk, kk, vk, ok, bk)
    size = ctypes.c_size_t(0)
    lib.check(lib.fn["varlen_decode_workspace_bytes"](sequences, q_heads, kv_heads, max_blocks, dv,
                                                      ctypes.byref(size)), "provider_preparation")
    workspace = torch.empty(max(size.value, 1), dtype=torch.uint8, device=device)
    keep += [strides, workspace]
    fn = lib.fn["varlen_decode_sink"]
    args = (qk.data_ptr(), kk.data_ptr(), vk.data_ptr(), cuk.data_ptr(), sk.data_ptr(), ok.data_ptr(), bk.data_ptr(),
            sequences, rows, q_heads, kv_heads, group, d, dv, max_blocks, strides, float(scale),
            workspace.data_ptr(), size.value)
    return Launch("intent_hip_varlen_decode_sink", lambda stream: fn(*args, stream), tuple(keep), tuple(before),
                  tuple(after), (("sequences", sequences), ("rows", rows), ("q_heads", q_heads),
                                 ("kv_heads", kv_heads), ("d", d), ("max_blocks", max_blocks),
                                 ("workspace_bytes", size.value)),
                  lambda: lib.kernel_resources(OP_VARLEN_DECODE, F16, group, d))


def _splitk_reduce(lib, bound, constexprs, device):
    partial, lse, output = bound.arguments
    keep, before, after = [partial, lse, output], [], []
    pk, outk = _readable(partial, keep, before), _writable(output, keep, after)
    batch, heads, splits, d = partial.shape
    strides = _strides(pk, lse, outk)
    keep.append(strides)
    fn = lib.fn["splitk_reduce_f32_to_f16"]
    args = (pk.data_ptr(), lse.data_ptr(), outk.data_ptr(), batch, heads, splits, d, strides)
    return Launch("intent_hip_splitk_reduce_f32_to_f16", lambda stream: fn(*args, stream), tuple(keep),
                  tuple(before), tuple(after),
                  (("batch", batch), ("heads", heads), ("splits", splits), ("d", d)),
                  lambda: lib.kernel_resources(OP_SPLITK_REDUCE, F32, batch * heads, d))


# ------------------------------------------------------------------------------ SpMV
def _csr_spmv(lib, bound, constexprs, device):
    import ctypes

    import torch

    offsets, columns, values, vector, output = bound.arguments
    rows = offsets.shape[0] - 1
    if rows < 0 or output.shape[0] != rows:
        raise ValueError("csr_spmv requires row_offsets.shape[0] == output.shape[0] + 1")
    if columns.shape[0] != values.shape[0]:
        raise ValueError("csr_spmv requires column_indices and values of equal length")
    keep, before, after = [offsets, columns, values, vector, output], [], []
    ok, ck, vk, xk, yk = (_readable(offsets, keep, before), _readable(columns, keep, before),
                          _readable(values, keep, before), _readable(vector, keep, before),
                          _writable(output, keep, after))
    nnz, cols = values.shape[0], vector.shape[0]
    size = ctypes.c_size_t(0)
    lib.check(lib.fn["csr_spmv_workspace_bytes"](rows, nnz, ctypes.byref(size)), "provider_preparation")
    pointers = (ok.data_ptr(), ck.data_ptr(), vk.data_ptr(), xk.data_ptr(), yk.data_ptr(), rows, cols, nnz)
    facts = (("rows", rows), ("cols", cols), ("nnz", nnz), ("workspace_bytes", size.value))
    if _static_workspace():
        if size.value > STATIC_SCRATCH_BYTES:
            raise CompilationStageError(
                "provider_preparation", f"csr_spmv of {rows} rows and {nnz} nonzeros needs {size.value} workspace "
                f"bytes, beyond the {STATIC_SCRATCH_BYTES}-byte static scratch; use workspace='prepare'")
        fn, entry = lib.fn["csr_spmv_f32_static"], "intent_hip_csr_spmv_f32_static"
        args = pointers
        facts += (("workspace", "static"),)
    else:
        workspace = torch.empty(max(size.value, 1), dtype=torch.uint8, device=device)
        keep.append(workspace)
        fn, entry = lib.fn["csr_spmv_f32"], "intent_hip_csr_spmv_f32"
        args = (*pointers, workspace.data_ptr(), size.value)
    return Launch(entry, lambda stream: fn(*args, stream), tuple(keep), tuple(before), tuple(after), facts,
                  lambda: lib.kernel_resources(OP_CSR_SPMV_F32, F32, rows, nnz))


def _csr_spmm(lib, bound, constexprs, device):
    """csr_spmm: rows read through their own strides (unit inner stride required, staged otherwise)."""
    offsets, columns, values, dense, output = bound.arguments
    rows = offsets.shape[0] - 1
    if rows < 0 or output.shape[0] != rows:
        raise ValueError("csr_spmm requires row_offsets.shape[0] == output.shape[0] + 1")
    if columns.shape[0] != values.shape[0]:
        raise ValueError("csr_spmm requires column_indices and values of equal length")
    if dense.shape[1] != output.shape[1]:
        raise ValueError("csr_spmm requires dense and output of equal feature width")
    keep, before, after = [offsets, columns, values, dense, output], [], []
    ok, ck, vk = (_readable(offsets, keep, before), _readable(columns, keep, before), _readable(values, keep, before))
    dk, outk = _readable(dense, keep, before), _writable(output, keep, after)
    nnz, cols, features = values.shape[0], dense.shape[0], dense.shape[1]
    fn = lib.fn["csr_spmm_f32"]
    args = (ok.data_ptr(), ck.data_ptr(), vk.data_ptr(), dk.data_ptr(), outk.data_ptr(), rows, cols, nnz, features,
            _row_stride(dk) if cols else features, _row_stride(outk) if rows else features)
    return Launch("intent_hip_csr_spmm_f32", lambda stream: fn(*args, stream), tuple(keep), tuple(before),
                  tuple(after), (("rows", rows), ("cols", cols), ("nnz", nnz), ("features", features)),
                  lambda: lib.kernel_resources(OP_CSR_SPMM_F32, F32, rows, features))


def _no_static(name, use):
    if _static_workspace():
        raise CompilationStageError("provider_preparation", f"{name} {use} a workspace; backend_options workspace='static' has "
                                    "none for it, use workspace='prepare'")


# ------------------------------------------------------------------------------ norm and rotation of heads
def _interleaved(constexprs) -> int:
    value = constexprs["INTERLEAVED"]
    if not isinstance(value, bool):
        raise CompilationStageError("provider_configuration", f"INTERLEAVED must be a bool, got {value!r}")
    return int(value)


def _norm_rope_staged(arguments, extents, outputs):
    """(the arguments with the views that the kernels take in place of those they do not, what is copied before and after)"""
    tokens, _, _, d, table, pairs = extents
    if 2 * pairs > d:
        raise ValueError(f"{pairs} rotated pairs do not fit heads of width {d}")
    if pairs and not table and tokens:
        raise ValueError("the rotation tables hold no position")
    keep, before, after = [], [], []
    last = len(arguments) - 1
    values = [_readable(t, keep, before) for t in arguments[:last - outputs]]
    values += [_writable(t, keep, after) for t in arguments[last - outputs:last]]
    return (*values, arguments[last]), before, after


def _norm_rope_mixed(values, last) -> int:
    """`_mixed` of the rows, of the weights of the heads there are, and of the tables; `last`: the last view of rows."""
    weights = [w for x, w in zip(values[:2], values[2:4]) if x.numel()]
    return _mixed(*values[:2], *weights, *values[5:last + 1])


def _norm_rope_extents(q, k, cos) -> tuple:
    return (q.shape[0], q.shape[1], k.shape[1], q.shape[2], *cos.shape)


def _mixed(*views) -> int:
    """Every address, and every outer stride in bytes, or-ed: what the views' common alignment can be read from."""
    mixed = 0
    for t in views:
        if t.numel():
            mixed |= t.data_ptr()
            for st in t.stride()[:-1]:
                mixed |= st * t.element_size()
    return mixed


_NORM_ROPE_EXTENTS = ("tokens", "q_heads", "kv_heads", "d", "table", "pairs")


def _norm_rope(dtype_code):
    """qk_norm_rope: q and k rows are read through their own strides (a projection's slices), staged only where their
    inner stride is not 1."""
    def plan(lib, bound, constexprs, device):
        interleaved = _interleaved(constexprs)
        extents = _norm_rope_extents(bound.arguments[0], bound.arguments[1], bound.arguments[5])
        values, before, after = _norm_rope_staged(bound.arguments, extents, 2)
        strides = _strides(*values[:2], *values[5:9])
        fn, configuration = lib.fn["qk_norm_rope"], tuple(zip(_NORM_ROPE_EXTENTS, extents))

        def again(values):
            args = (dtype_code, *[t.data_ptr() for t in values[:9]], *extents, strides, float(values[9]), interleaved)
            return Launch("intent_hip_qk_norm_rope", lambda stream: fn(*args, stream), values, configuration=configuration,
                          resources=lambda: lib.call_resources(OP_QK_NORM_ROPE, dtype_code, extents[3], extents[5], interleaved,
                                                               _norm_rope_mixed(values, 8)))
        return _staged(again, values, bound, before, after)
    return plan


def _norm_rope_backward(dtype_code):
    """qk_norm_rope_backward: workgroups keep their share of the weights' gradients, summed in order through a workspace."""
    def plan(lib, bound, constexprs, device):
        import ctypes

        interleaved = _interleaved(constexprs)
        extents = _norm_rope_extents(bound.arguments[0], bound.arguments[1], bound.arguments[5])
        _no_static("qk_norm_rope_backward", "sums the weights' gradients through")
        values, before, after = _norm_rope_staged(bound.arguments, extents, 4)
        strides = _strides(*values[:2], *values[5:11])
        size = ctypes.c_size_t(0)
        lib.check(lib.fn["qk_norm_rope_backward_workspace_bytes"](*extents[:4], ctypes.byref(size)), "provider_preparation")
        fn, size = lib.fn["qk_norm_rope_backward"], size.value
        configuration = (*zip(_NORM_ROPE_EXTENTS, extents), ("workspace_bytes", size))

        def again(values):
            args = (dtype_code, *[t.data_ptr() for t in values[:13]], *extents, strides, float(values[13]), interleaved)
            keep = [values]
            run = _workspace_run(fn, args, size, device, keep)
            return Launch("intent_hip_qk_norm_rope_backward", run, tuple(keep), configuration=configuration,
                          resources=lambda: lib.call_resources(OP_QK_NORM_ROPE_BACKWARD, dtype_code, extents[3], extents[5],
                                                               interleaved, _norm_rope_mixed(values, 10)))
        return _staged(again, values, bound, before, after)
    return plan


def _norm_rope_signature(element, backward):
    rows, table, weight = _view(IN, element, 3), _view(IN, "f32", 2), _view(IN, "f32", 1)
    inputs = (rows, rows, weight, weight, _view(IN, "i32", 1), table, table)
    out, out_weight = _view(OUT, element, 3), _view(OUT, "f32", 1)
    if backward:
        return (*inputs, rows, rows, out, out, out_weight, out_weight, ("scalar", "f32"))
    return (*inputs, out, out, ("scalar", "f32"))


# ------------------------------------------------------------------------------ paged cache of 8 bits
_MX_BLOCK = 32


def _cache_strides(name, elements, exponents) -> tuple:
    """The strides of a cache's elements and exponents as the kernels take them (0 along an axis of one). A cache is never
    staged: its pages are read, and written, in place."""
    width = elements.shape[3]
    if width % _MX_BLOCK or exponents.shape[3] * _MX_BLOCK != width:
        raise ValueError(f"{name} rows are blocks of {_MX_BLOCK} elements with one exponent each; got widths {width} and "
                         f"{exponents.shape[3]}")
    if elements.numel() and not _aligned(elements, 16):
        raise ValueError(f"{name} elements need unit inner stride, other strides in multiples of 16 and a 16-byte aligned "
                         f"start, got strides {tuple(elements.stride())}")
    if not _aligned(exponents, 1):
        raise ValueError(f"{name} exponents need unit inner stride, got strides {tuple(exponents.stride())}")
    return (*_outer_strides(elements), 1, *_outer_strides(exponents), 1)


def _outer_strides(tensor) -> tuple:
    return tuple(st if n > 1 else 0 for st, n in zip(tensor.stride()[:-1], tensor.shape[:-1]))


def _paged_cache(dtype_code, reading: bool):
    """paged_cache_append / paged_cache_read: the same tables and strides, the rows read or written."""
    def plan(lib, bound, constexprs, device):
        import ctypes

        if reading:
            *cache, cu, page_offsets, page_indices, k, v = bound.arguments
        else:
            k, v, *cache, cu, page_offsets, page_indices, lengths = bound.arguments
            if lengths.shape[0] + 1 != cu.shape[0]:
                raise ValueError(f"cu_seqlens and page_offsets need sequence_lengths.shape[0] + 1 = {lengths.shape[0] + 1} "
                                 f"entries, got {cu.shape[0]}")
        if cu.shape[0] < 1:
            raise ValueError("cu_seqlens needs an entry per sequence and one more")
        keep, before, after = [], [], []
        held = (*_cache_strides("key", *cache[:2]), *_cache_strides("value", *cache[2:]))
        rows = [_writable(t, keep, after, 8) if reading else _readable(t, keep, before, 8) for t in (k, v)]
        if reading and after:      # a staged output starts as the caller's, whose rows behind the last sequence stay
            before += [functools.partial(staged.copy_, out) for staged, out in zip(rows, (k, v)) if staged is not out]
        strides = (ctypes.c_int64 * 22)(*(x for t in rows for x in (*_outer_strides(t), 1)), *held)
        tables = [_readable(t, keep, before) for t in (cu, page_offsets, page_indices)]
        pages, ps, kv_heads, d = cache[0].shape
        extents = (k.shape[0], cu.shape[0] - 1, kv_heads, d, cache[2].shape[3], pages, ps, page_indices.shape[0])
        configuration = tuple(zip(("rows", "sequences", "kv_heads", "d", "dv", "pages", "ps", "positions"), extents))
        if reading:
            fn, entry, op = lib.fn["paged_cache_read"], "intent_hip_paged_cache_read", OP_PAGED_CACHE_READ
            values = (*cache, *tables, *rows)
        else:
            fn, entry, op = lib.fn["paged_cache_append"], "intent_hip_paged_cache_append", OP_PAGED_CACHE_APPEND
            values = (*rows, *cache, *tables, _readable(lengths, keep, before))

        def again(values):
            args = (dtype_code, *[t.data_ptr() for t in values], *extents, strides)
            return Launch(entry, lambda stream: fn(*args, stream), values, configuration=configuration,
                          resources=lambda: lib.kernel_resources(op, dtype_code, extents[0], extents[2] * (extents[3] + extents[4])))
        return _staged(again, values, bound, before, after)
    return plan


def _paged_decode_mx(dtype_code):
    """paged_gqa_decode_mx: jobs of a sequence's pages, whose states a second kernel joins through a workspace; none where
    one job holds every page."""
    def plan(lib, bound, constexprs, device):
        import ctypes

        q, *cache, page_offsets, page_indices, lengths, output, scale = bound.arguments
        group = _positive_constexpr(constexprs, "HEAD_GROUP")
        batch, q_heads, d = q.shape
        pages, ps, kv_heads, _ = cache[0].shape
        if kv_heads * group != q_heads:
            raise ValueError(f"query heads ({q_heads}) must equal key/value heads ({kv_heads}) * HEAD_GROUP ({group})")
        if page_offsets.shape[0] != batch + 1:
            raise ValueError(f"page_offsets must hold batch + 1 = {batch + 1} entries, got {page_offsets.shape[0]}")
        keep, before, after = [], [], []
        held = (*_cache_strides("key", *cache[:2]), *_cache_strides("value", *cache[2:]))
        q, output = _readable(q, keep, before, 8), _writable(output, keep, after)
        tables = [_readable(t, keep, before) for t in (page_offsets, page_indices, lengths)]
        strides = (ctypes.c_int64 * 22)(*_outer_strides(q), 1, *held, *_outer_strides(output), 1)
        reach = max(held[1], held[5], held[9], held[13])         # the tokens' strides
        positions, size = page_indices.shape[0], ctypes.c_size_t(0)
        lib.check(lib.fn["paged_gqa_decode_mx_workspace_bytes"](batch, q_heads, kv_heads, group, d, ps, positions,
                                                                ctypes.byref(size)), "provider_preparation")
        fn, size = lib.fn["paged_gqa_decode_mx"], size.value
        if size:
            _decode_workspace("paged_gqa_decode_mx")
        configuration = (("batch", batch), ("q_heads", q_heads), ("kv_heads", kv_heads), ("d", d), ("pages", pages), ("ps", ps),
                         ("positions", positions), ("workspace_bytes", size))

        def again(values):
            args = (dtype_code, *[t.data_ptr() for t in values[:9]], batch, q_heads, kv_heads, group, d, pages, ps, positions,
                    strides, float(values[9]))
            keep = [values]
            return Launch("intent_hip_paged_gqa_decode_mx", _optional_workspace_run(fn, args, size, device, keep), tuple(keep),
                          configuration=configuration,
                          resources=lambda: lib.call_resources(OP_PAGED_GQA_DECODE_MX, dtype_code, batch, kv_heads, group, d, ps,
                                                               positions, reach))
        return _staged(again, (q, *cache, *tables, output, scale), bound, before, after)
    return plan


def _cache_signature(access):
    elements, exponents = _view(access, "f8e4m3fn", 4), _view(access, "u8", 4)
    return (elements, exponents, elements, exponents)


def _append_signature(element):
    rows, table = _view(IN, element, 3), _view(IN, "i32", 1)
    return (rows, rows, *_cache_signature(INOUT), table, table, table, table)


def _read_signature(element):
    rows, table = _view(OUT, element, 3), _view(IN, "i32", 1)
    return (*_cache_signature(IN), table, table, table, rows, rows)


def _decode_mx_signature(element):
    rows, table = _view(IN, element, 3), _view(IN, "i32", 1)
    return (rows, *_cache_signature(IN), table, table, table, _view(OUT, element, 3), ("scalar", "f32"))


# ------------------------------------------------------------------------------ 4-bit weights
def _linear_mxfp4(dtype_code):
    """linear_mxfp4: x is staged where its layout is not the kernel's; a weight never is."""
    def plan(lib, bound, constexprs, device):
        import ctypes

        x, weight, exponents, out = bound.arguments
        (m, k), n = x.shape, weight.shape[0]
        if k % _MX_BLOCK or weight.shape[1] * 2 != k or exponents.shape[1] * _MX_BLOCK != k:
            raise ValueError(f"weights of K = {k} are blocks of {_MX_BLOCK} elements: [N, K / 2] bytes and [N, K / {_MX_BLOCK}] "
                             f"exponents, got {tuple(weight.shape)} and {tuple(exponents.shape)}")
        if not _aligned(weight, 16) or not _aligned(exponents, 1):
            raise ValueError(f"weights need unit inner stride, rows in multiples of 16 bytes and a 16-byte aligned start, and "
                             f"their exponents unit inner stride; got strides {tuple(weight.stride())} and "
                             f"{tuple(exponents.stride())}")
        keep, before, after = [], [], []
        x, out = _readable(x, keep, before, 8), _writable(out, keep, after)
        extents = (m, n, k, *(_outer_strides(t)[0] for t in (x, weight, exponents, out)))
        size = ctypes.c_size_t(0)
        lib.check(lib.fn["linear_mxfp4_workspace_bytes"](m, n, k, ctypes.byref(size)), "provider_preparation")
        fn, size = lib.fn["linear_mxfp4"], size.value
        if size:
            _no_static("linear_mxfp4", "divides K of few tiles over workgroups whose sums meet in")
        configuration = (("m", m), ("n", n), ("k", k), ("workspace_bytes", size))

        def again(values):
            args = (dtype_code, *[t.data_ptr() for t in values], *extents)
            keep = [values]
            return Launch("intent_hip_linear_mxfp4", _optional_workspace_run(fn, args, size, device, keep), tuple(keep),
                          configuration=configuration, resources=lambda: lib.call_resources(OP_LINEAR_MXFP4, dtype_code, m, n, k))
        return _staged(again, (x, weight, exponents, out), bound, before, after)
    return plan


# ------------------------------------------------------------------------------ norm of the residual stream
def _residual_norm_checked(gate, post_weight, weight, tokens):
    """(number of gates, of the block's norm's weights), each 0 where there is none."""
    gates, post, d = gate.shape[0], post_weight.shape[0], weight.shape[0]
    if gates not in (0, tokens):
        raise ValueError(f"gate holds a number for each of {tokens} tokens, or none at all; got {gates}")
    if post not in (0, d):
        raise ValueError(f"post_weight holds a number for each of {d} columns, or none at all; got {post}")
    return gates, post


def _rows_mixed(wide, narrow=()) -> int:
    """`_mixed` of rows of 16 bits and of weights, and of rows of 8 bits at twice their size: pieces of 16 and of 8 bytes."""
    return _mixed(*wide) | 2 * _mixed(*narrow)


def _residual_norm(dtype_code, narrow: bool):
    """residual_norm, residual_norm_i8: rows are read through their own strides, staged only where their inner stride is not 1."""
    name = "residual_norm_i8" if narrow else "residual_norm"

    def plan(lib, bound, constexprs, device):
        import ctypes

        block, residual, gate, post_weight, weight, total, output, *more = bound.arguments
        scales, numbers = more[:-3], more[-3:]
        (tokens, d), (gates, post) = block.shape, _residual_norm_checked(gate, post_weight, weight, block.shape[0])
        keep, before, after = [], [], []
        block, residual, post_weight, weight = (_readable(t, keep, before) for t in (block, residual, post_weight, weight))
        total, output, *scales = (_writable(t, keep, after) for t in (total, output, *scales))
        strides = (ctypes.c_int64 * 5)(*(t.stride(0) for t in (block, residual, gate, total, output)))
        fn, op = lib.fn[name], OP_RESIDUAL_NORM_I8 if narrow else OP_RESIDUAL_NORM
        configuration = (("tokens", tokens), ("d", d), ("gates", gates), ("post", post))

        def again(values):
            args = (dtype_code, *[t.data_ptr() for t in values[:-3]], tokens, d, gates, post, strides, *map(float, values[-3:]))
            rows = (*values[:2], *values[3:6])
            return Launch("intent_hip_" + name, lambda stream: fn(*args, stream), values, configuration=configuration,
                          resources=lambda: lib.call_resources(op, dtype_code, d, post, _rows_mixed(rows, values[6:7]) if narrow
                                                               else _rows_mixed((*rows, values[6]))))
        return _staged(again, (block, residual, gate, post_weight, weight, total, output, *scales, *numbers), bound, before, after)
    return plan


def _residual_norm_backward(dtype_code):
    """residual_norm_backward: each slot of tokens keeps its share of the weights' gradients, summed in order through a workspace."""
    def plan(lib, bound, constexprs, device):
        import ctypes

        block, total, gate, post_weight, weight, *rest = bound.arguments
        grads, (grad_block, grad_residual, grad_gate, *grad_weights), numbers = rest[:2], rest[2:7], rest[7:]
        (tokens, d), (gates, post) = block.shape, _residual_norm_checked(gate, post_weight, weight, block.shape[0])
        _no_static("residual_norm_backward", "sums the weights' gradients through")
        keep, before, after = [], [], []
        block, total, post_weight, weight, *grads = (_readable(t, keep, before) for t in (block, total, post_weight, weight, *grads))
        grad_block, grad_residual, *grad_weights = (_writable(t, keep, after) for t in (grad_block, grad_residual, *grad_weights))
        strides = (ctypes.c_int64 * 8)(*(t.stride(0) for t in (block, total, gate, *grads, grad_block, grad_residual, grad_gate)))
        size = ctypes.c_size_t(0)
        lib.check(lib.fn["residual_norm_backward_workspace_bytes"](tokens, d, post, ctypes.byref(size)), "provider_preparation")
        fn, size = lib.fn["residual_norm_backward"], size.value
        configuration = (("tokens", tokens), ("d", d), ("gates", gates), ("post", post), ("workspace_bytes", size))

        def again(values):
            args = (dtype_code, *[t.data_ptr() for t in values[:12]], tokens, d, gates, post, strides, *map(float, values[12:]))
            keep = [values]
            return Launch("intent_hip_residual_norm_backward", _optional_workspace_run(fn, args, size, device, keep), tuple(keep),
                          configuration=configuration,
                          resources=lambda: lib.call_resources(OP_RESIDUAL_NORM_BACKWARD, dtype_code, d, post,
                                                               _rows_mixed((*values[:2], *values[3:9]))))
        return _staged(again, (block, total, gate, post_weight, weight, *grads, grad_block, grad_residual, grad_gate, *grad_weights,
                               *numbers), bound, before, after)
    return plan


def _residual_norm_signature(element, kind):
    rows, weight, number = _view(IN, element, 2), _view(IN, "f32", 1), ("scalar", "f32")
    out, out_weight = _view(OUT, element, 2), _view(OUT, "f32", 1)
    if kind == "backward":
        return (rows, rows, *[weight] * 3, rows, rows, out, out, *[out_weight] * 3, *[number] * 3)
    outputs = (out, _view(OUT, "i8", 2), out_weight) if kind == "i8" else (out, out)
    return (rows, rows, *[weight] * 3, *outputs, *[number] * 3)


# Rows that may be written where rows were read, each element by the thread that read it: sum and output over block and residual
# (8-bit rows are others), gradients over any rows.
_NORM_IN_PLACE = frozenset(((0, 5), (1, 5), (0, 6), (1, 6)))
_NORM_I8_IN_PLACE = frozenset(((0, 5), (1, 5)))
_NORM_BACKWARD_IN_PLACE = frozenset((i, j) for i in (0, 1, 5, 6) for j in (7, 8))


# ------------------------------------------------------------------------------ products of 8-bit integers
def _quantize_rows(dtype_code, gated: bool):
    """quantize_rows, swiglu_quantize_rows: rows (halves of one projection's, say) are read through their own strides."""
    name, op = ("swiglu_quantize_rows", OP_SWIGLU_QUANTIZE_ROWS) if gated else ("quantize_rows", OP_QUANTIZE_ROWS)

    def plan(lib, bound, constexprs, device):
        *rows, output, scales = bound.arguments
        keep, before, after = [], [], []
        rows = [_readable(t, keep, before) for t in rows]
        output, scales = (_writable(t, keep, after) for t in (output, scales))
        count, d = output.shape
        strides = tuple(t.stride(0) for t in (*rows, output))
        fn = lib.fn[name]

        def again(values):
            args = (dtype_code, *[t.data_ptr() for t in values], count, d, *strides)
            return Launch("intent_hip_" + name, lambda stream: fn(*args, stream), values, configuration=(("rows", count), ("d", d)),
                          resources=lambda: lib.call_resources(op, dtype_code, d, _rows_mixed(values[:-2], values[-2:-1])))
        return _staged(again, (*rows, output, scales), bound, before, after)
    return plan


def _quantize_rows_signature(element, gated):
    return (*[_view(IN, element, 2)] * (2 if gated else 1), _view(OUT, "i8", 2), _view(OUT, "f32", 1))


def _linear_i8(dtype_code):
    """linear_i8: x is staged where its layout is not the kernel's; a weight never is."""
    def plan(lib, bound, constexprs, device):
        import ctypes

        x, weight, x_scales, weight_scales, bias, out = bound.arguments
        (m, k), n, biases = x.shape, weight.shape[0], bias.shape[0]
        if k % 16:
            raise ValueError(f"products of 8-bit integers take K in multiples of 16, got {k}")
        if biases not in (0, n):
            raise ValueError(f"bias holds a number for each of {n} columns, or none at all; got {biases}")
        if not _aligned(weight, 16):
            raise ValueError(f"weights need unit inner stride, rows in multiples of 16 bytes and a 16-byte aligned start; got strides "
                             f"{tuple(weight.stride())}")
        keep, before, after = [], [], []
        x, out = _readable(x, keep, before, 16), _writable(out, keep, after)
        x_scales, weight_scales, bias = (_readable(t, keep, before) for t in (x_scales, weight_scales, bias))
        extents = (m, n, k, *(_outer_strides(t)[0] for t in (x, weight, out)))
        size = ctypes.c_size_t(0)
        lib.check(lib.fn["linear_i8_workspace_bytes"](m, n, k, ctypes.byref(size)), "provider_preparation")
        fn, size = lib.fn["linear_i8"], size.value
        if size:
            _no_static("linear_i8", "divides K of few tiles over workgroups whose sums meet in")
        configuration = (("m", m), ("n", n), ("k", k), ("bias", biases > 0), ("workspace_bytes", size))

        def again(values):
            addresses = [t.data_ptr() for t in values]
            if not biases:
                addresses[4] = None
            args = (dtype_code, *addresses, *extents)
            keep = [values]
            return Launch("intent_hip_linear_i8", _optional_workspace_run(fn, args, size, device, keep), tuple(keep),
                          configuration=configuration, resources=lambda: lib.call_resources(OP_LINEAR_I8, dtype_code, m, n, k))
        return _staged(again, (x, weight, x_scales, weight_scales, bias, out), bound, before, after)
    return plan


def _linear_i8_signature(element):
    return (_view(IN, "i8", 2), _view(IN, "i8", 2), *[_view(IN, "f32", 1)] * 3, _view(OUT, element, 2))


# ------------------------------------------------------------------------------ decode behind a shared prefix
def _paged_decode_prefix(dtype_code):
    """paged_gqa_decode_prefix: parts of the prefix and jobs of the sequences' pages, whose states a second kernel joins through a
    workspace. The caches are read in place, never staged."""
    def plan(lib, bound, constexprs, device):
        import ctypes

        q, *caches, prefix_indices, prefix_length, page_offsets, page_indices, lengths, output, scale = bound.arguments
        group = _positive_constexpr(constexprs, "HEAD_GROUP")
        batch, q_heads, d = q.shape
        pages, ps, kv_heads, _ = caches[0].shape
        if kv_heads * group != q_heads:
            raise ValueError(f"query heads ({q_heads}) must equal key/value heads ({kv_heads}) * HEAD_GROUP ({group})")
        if prefix_length.shape[0] != 1:
            raise ValueError(f"prefix_length holds one number, got {prefix_length.shape[0]}")
        if page_offsets.shape[0] != batch + 1:
            raise ValueError(f"page_offsets must hold batch + 1 = {batch + 1} entries, got {page_offsets.shape[0]}")
        for name, cache in zip(("key_cache", "value_cache"), caches):
            if not _aligned(cache, 8):
                raise ValueError(f"{name} needs unit inner stride, other strides in multiples of 8 and a 16-byte aligned start, got "
                                 f"strides {tuple(cache.stride())}")
        _no_static("paged_gqa_decode_prefix", "joins the states of its jobs through")
        keep, before, after = [], [], []
        q, output = _readable(q, keep, before, 8), _writable(output, keep, after)
        tables = [_readable(t, keep, before) for t in (prefix_indices, prefix_length, page_offsets, page_indices, lengths)]
        strides = (ctypes.c_int64 * 14)(*(st for t in (q, *caches, output) for st in (*_outer_strides(t), 1)))
        extents, reach = (batch, q_heads, kv_heads, group, d), max(strides[3], strides[7], strides[4] * ps, strides[8] * ps)
        positions, size = (prefix_indices.shape[0], page_indices.shape[0]), ctypes.c_size_t(0)
        lib.check(lib.fn["paged_gqa_decode_prefix_workspace_bytes"](*extents, ps, *positions, ctypes.byref(size)),
                  "provider_preparation")
        fn, size = lib.fn["paged_gqa_decode_prefix"], size.value
        configuration = (("batch", batch), ("q_heads", q_heads), ("kv_heads", kv_heads), ("d", d), ("pages", pages), ("ps", ps),
                         ("prefix_positions", positions[0]), ("positions", positions[1]), ("workspace_bytes", size))

        def again(values):
            args = (dtype_code, *[t.data_ptr() for t in values[:9]], *extents, pages, ps, *positions, strides, float(values[9]))
            keep = [values]
            return Launch("intent_hip_paged_gqa_decode_prefix", _optional_workspace_run(fn, args, size, device, keep), tuple(keep),
                          configuration=configuration,
                          resources=lambda: lib.call_resources(OP_PAGED_GQA_DECODE_PREFIX, dtype_code, batch, kv_heads, group, d, ps,
                                                               *positions, reach))
        return _staged(again, (q, *caches, *tables, output, scale), bound, before, after)
    return plan


def _decode_prefix_signature(element):
    rows, cache, table = _view(IN, element, 3), _view(IN, element, 4), _view(IN, "i32", 1)
    return (rows, cache, cache, *[table] * 5, _view(OUT, element, 3), ("scalar", "f32"))


_repeated = functools.partial(OperatorSpec, repeats=True)
_SPECS = (
    OperatorSpec("stable_softmax", (_view(IN, "f32", 2), _view(OUT, "f32", 2)), (), _softmax_fwd(F32), True),
    OperatorSpec("stable_softmax_f16", (_view(IN, "f16", 2), _view(OUT, "f16", 2)), (), _softmax_fwd(F16), True),
    OperatorSpec("chunked_softmax_bf16", (_view(IN, "bf16", 2), _view(OUT, "bf16", 2)), (), _softmax_fwd(BF16),
                 True),
    OperatorSpec("softmax_backward", (_view(IN, "f32", 2), _view(IN, "f32", 2), _view(OUT, "f32", 2)), (),
                 _softmax_bwd(F32), True),
    OperatorSpec("softmax_backward_f16", (_view(IN, "f16", 2), _view(IN, "f16", 2), _view(OUT, "f16", 2)), (),
                 _softmax_bwd(F16), True),
    OperatorSpec("gemm_f32", (_view(IN, "f32", 2), _view(IN, "f32", 2), _view(OUT, "f32", 2)), (),
                 _gemm_f32(False)),
    OperatorSpec("linear_f32", (_view(IN, "f32", 2), _view(IN, "f32", 2), _view(OUT, "f32", 2)), (),
                 _gemm_f32(True)),
    OperatorSpec("gemm_i8", (_view(IN, "i8", 2), _view(IN, "i8", 2), _view(IN, "i32", 1), _view(OUT, "i32", 2)), (),
                 _gemm_i8),
    OperatorSpec("gemm", (_view(IN, "f16", 2), _view(IN, "f16", 2), _view(OUT, "f16", 2)), ("ACTIVATION",),
                 _gemm16(F16)),
    OperatorSpec("quantized_gemm", (_view(IN, "f16", 2), _view(IN, "f16", 2), _view(IN, "f32", 1), _view(IN, "f16", 2),
                                    _view(IN, "f32", 1), _view(OUT, "i8", 2)), (), _quantized_gemm),
    OperatorSpec("bf16_gemm", (_view(IN, "bf16", 2), _view(IN, "bf16", 2), _view(OUT, "bf16", 2)), (),
                 _gemm_bf16),
    OperatorSpec("flash_attention_fwd", (_view(IN, "f16", 4), _view(IN, "f16", 4), _view(IN, "f16", 4),
                                         _view(OUT, "f16", 4), ("scalar", "f32")), ("CAUSAL",), _attention_f16),
    OperatorSpec("flash_gqa_attention_fwd", (_view(IN, "f16", 4), _view(IN, "f16", 4), _view(IN, "f16", 4),
                                             _view(OUT, "f16", 4), ("scalar", "f32")), ("HEAD_GROUP", "CAUSAL"),
                 _attention_grouped(F16)),
    OperatorSpec("flash_attention_bf16_fwd", (_view(IN, "bf16", 4), _view(IN, "bf16", 4), _view(IN, "bf16", 4),
                                              _view(OUT, "bf16", 4), ("scalar", "f32")), ("HEAD_GROUP", "CAUSAL"),
                 _attention_grouped(BF16)),
    OperatorSpec("mla_prefill", (_view(IN, "f16", 4), _view(IN, "f16", 4), _view(IN, "f16", 4), _view(IN, "f16", 4),
                                 _view(IN, "f16", 4), _view(OUT, "f16", 4), ("scalar", "f32")), ("HEAD_GROUP",),
                 _mla_prefill),
    OperatorSpec("flash_attention_bias_fwd", (_view(IN, "f16", 4), _view(IN, "f16", 4), _view(IN, "f16", 4),
                                              _view(IN, "f32", 3), _view(OUT, "f16", 4), ("scalar", "f32")), (),
                 _attention_bias),
    OperatorSpec("flash_varlen_attention_fwd",
                 (_view(IN, "f16", 2), _view(IN, "f16", 2), _view(IN, "f16", 2), _view(IN, "i32", 1),
                  _view(IN, "i32", 1), _view(OUT, "f16", 2), ("scalar", "f32")), ("CAUSAL",),
                 _attention_varlen(False)),
    OperatorSpec("flash_varlen_gqa_prefill",
                 (_view(IN, "f16", 3), _view(IN, "f16", 3), _view(IN, "f16", 3), _view(IN, "i32", 1),
                  _view(IN, "i32", 1), _view(OUT, "f16", 3), ("scalar", "f32")), ("HEAD_GROUP",),
                 _attention_varlen(True)),
    OperatorSpec("attention_backward_delta", (_view(IN, "f16", 4), _view(IN, "f16", 4), _view(OUT, "f32", 3)), (),
                 _attention_bwd_delta),
    OperatorSpec("attention_backward_dkdv",
                 (_view(IN, "f16", 4), _view(IN, "f16", 4), _view(IN, "f16", 4), _view(IN, "f16", 4),
                  _view(IN, "f32", 3), _view(IN, "f32", 3), _view(OUT, "f16", 4), _view(OUT, "f16", 4),
                  ("scalar", "f32")), ("HEAD_GROUP", "CAUSAL"), _attention_bwd("dkdv")),
    OperatorSpec("attention_backward_dq",
                 (_view(IN, "f16", 4), _view(IN, "f16", 4), _view(IN, "f16", 4), _view(IN, "f16", 4),
                  _view(IN, "f32", 3), _view(IN, "f32", 3), _view(OUT, "f16", 4), ("scalar", "f32")),
                 ("HEAD_GROUP", "CAUSAL"), _attention_bwd("dq")),
    OperatorSpec("paged_gqa_decode_partials",
                 (_view(IN, "f16", 3), _view(IN, "f16", 4), _view(IN, "f16", 4), _view(IN, "i32", 1),
                  _view(IN, "i32", 1), _view(IN, "i32", 1), _view(IN, "i32", 1), _view(OUT, "f32", 3),
                  _view(OUT, "f32", 4), ("scalar", "f32")), ("PAGE_SIZE", "HEAD_GROUP", "SPLITS"),
                 _paged_decode_partials),
    OperatorSpec("grouped_flash_decode_partials",
                 (_view(IN, "bf16", 4), _view(IN, "bf16", 4), _view(IN, "bf16", 4), _view(OUT, "f32", 3),
                  _view(OUT, "bf16", 4), ("scalar", "f32")), ("HEAD_GROUP", "P", "SPLIT_SIZE"),
                 _grouped_decode_partials),
    OperatorSpec("continuous_gqa_decode",
                 (_view(IN, "f16", 3), _view(IN, "f16", 4), _view(IN, "f16", 4), _view(IN, "u8", 3),
                  _view(OUT, "f16", 3), ("scalar", "f32")), ("HEAD_GROUP",), _continuous_decode),
    OperatorSpec("varlen_gqa_decode_with_sink_logits",
                 (_view(IN, "f16", 3), _view(IN, "f16", 3), _view(IN, "f16", 3), _view(IN, "i32", 1),
                  _view(IN, "f32", 1), _view(OUT, "f16", 3), _view(OUT, "f32", 3), ("scalar", "f32")),
                 ("HEAD_GROUP", "MAX_BLOCKS"), _varlen_decode),
    OperatorSpec("splitk_attention_f32_to_f16_reduce", (_view(IN, "f32", 4), _view(IN, "f32", 3),
                                                        _view(OUT, "f16", 3)), (), _splitk_reduce),
    OperatorSpec("csr_spmm", (_view(IN, "i32", 1), _view(IN, "i32", 1), _view(IN, "f32", 1), _view(IN, "f32", 2),
                              _view(OUT, "f32", 2)), (), _csr_spmm, derived=(("R", "R1", -1),)),
    OperatorSpec("csr_spmv", (_view(IN, "i32", 1), _view(IN, "i32", 1), _view(IN, "f32", 1), _view(IN, "f32", 1),
                              _view(OUT, "f32", 1)), (), _csr_spmv, derived=(("R", "R1", -1),)),
    _repeated("qk_norm_rope_f16", _norm_rope_signature("f16", False), ("INTERLEAVED",), _norm_rope(F16)),
    _repeated("qk_norm_rope_bf16", _norm_rope_signature("bf16", False), ("INTERLEAVED",), _norm_rope(BF16)),
    _repeated("qk_norm_rope_backward_f16", _norm_rope_signature("f16", True), ("INTERLEAVED",), _norm_rope_backward(F16)),
    _repeated("qk_norm_rope_backward_bf16", _norm_rope_signature("bf16", True), ("INTERLEAVED",),
              _norm_rope_backward(BF16)),
    _repeated("paged_cache_append_f16", _append_signature("f16"), (), _paged_cache(F16, False)),
    _repeated("paged_cache_append_bf16", _append_signature("bf16"), (), _paged_cache(BF16, False)),
    _repeated("paged_cache_read_f16", _read_signature("f16"), (), _paged_cache(F16, True)),
    _repeated("paged_cache_read_bf16", _read_signature("bf16"), (), _paged_cache(BF16, True)),
    _repeated("paged_gqa_decode_mx_f16", _decode_mx_signature("f16"), ("HEAD_GROUP",), _paged_decode_mx(F16)),
    _repeated("paged_gqa_decode_mx_bf16", _decode_mx_signature("bf16"), ("HEAD_GROUP",), _paged_decode_mx(BF16)),
    _repeated("linear_mxfp4_f16", (_view(IN, "f16", 2), _view(IN, "u8", 2), _view(IN, "u8", 2), _view(OUT, "f16", 2)), (),
              _linear_mxfp4(F16)),
    _repeated("linear_mxfp4_bf16", (_view(IN, "bf16", 2), _view(IN, "u8", 2), _view(IN, "u8", 2), _view(OUT, "bf16", 2)), (),
              _linear_mxfp4(BF16)),
    _repeated("residual_norm_f16", _residual_norm_signature("f16", ""), (), _residual_norm(F16, False),
              inplace_safe=_NORM_IN_PLACE),
    _repeated("residual_norm_bf16", _residual_norm_signature("bf16", ""), (), _residual_norm(BF16, False),
              inplace_safe=_NORM_IN_PLACE),
    _repeated("residual_norm_i8_f16", _residual_norm_signature("f16", "i8"), (), _residual_norm(F16, True),
              inplace_safe=_NORM_I8_IN_PLACE),
    _repeated("residual_norm_i8_bf16", _residual_norm_signature("bf16", "i8"), (), _residual_norm(BF16, True),
              inplace_safe=_NORM_I8_IN_PLACE),
    _repeated("residual_norm_backward_f16", _residual_norm_signature("f16", "backward"), (), _residual_norm_backward(F16),
              inplace_safe=_NORM_BACKWARD_IN_PLACE),
    _repeated("residual_norm_backward_bf16", _residual_norm_signature("bf16", "backward"), (), _residual_norm_backward(BF16),
              inplace_safe=_NORM_BACKWARD_IN_PLACE),
    _repeated("quantize_rows_f16", _quantize_rows_signature("f16", False), (), _quantize_rows(F16, False)),
    _repeated("quantize_rows_bf16", _quantize_rows_signature("bf16", False), (), _quantize_rows(BF16, False)),
    _repeated("swiglu_quantize_rows_f16", _quantize_rows_signature("f16", True), (), _quantize_rows(F16, True)),
    _repeated("swiglu_quantize_rows_bf16", _quantize_rows_signature("bf16", True), (), _quantize_rows(BF16, True)),
    _repeated("linear_i8_f16", _linear_i8_signature("f16"), (), _linear_i8(F16)),
    _repeated("linear_i8_bf16", _linear_i8_signature("bf16"), (), _linear_i8(BF16)),
    _repeated("paged_gqa_decode_prefix_f16", _decode_prefix_signature("f16"), ("HEAD_GROUP",), _paged_decode_prefix(F16)),
    _repeated("paged_gqa_decode_prefix_bf16", _decode_prefix_signature("bf16"), ("HEAD_GROUP",), _paged_decode_prefix(BF16)),
)

SPECS = {spec.name: spec for spec in _SPECS}

ENTRY_POINTS = {
    "stable_softmax": "intent_hip_softmax_fwd", "stable_softmax_f16": "intent_hip_softmax_fwd",
    "chunked_softmax_bf16": "intent_hip_softmax_fwd", "softmax_backward": "intent_hip_softmax_bwd",
    "softmax_backward_f16": "intent_hip_softmax_bwd", "gemm_f32": "intent_hip_gemm_f32",
    "linear_f32": "intent_hip_gemm_f32", "gemm_i8": "intent_hip_gemm_i8", "gemm": "intent_hip_gemm",
    "quantized_gemm": "intent_hip_quantized_gemm", "bf16_gemm": "intent_hip_gemm_bf16",
    "flash_attention_fwd": "intent_hip_attention_fwd_f16", "flash_gqa_attention_fwd": "intent_hip_attention_fwd",
    "flash_attention_bf16_fwd": "intent_hip_attention_fwd", "mla_prefill": "intent_hip_mla_prefill",
    "flash_attention_bias_fwd": "intent_hip_attention_bias_fwd",
    "flash_varlen_attention_fwd": "intent_hip_attention_varlen_fwd",
    "flash_varlen_gqa_prefill": "intent_hip_attention_varlen_fwd",
    "attention_backward_delta": "intent_hip_attention_bwd_delta",
    "attention_backward_dkdv": "intent_hip_attention_bwd_dkdv", "attention_backward_dq": "intent_hip_attention_bwd_dq",
    "paged_gqa_decode_partials": "intent_hip_paged_decode_partials",
    "grouped_flash_decode_partials": "intent_hip_grouped_decode_partials",
    "continuous_gqa_decode": "intent_hip_continuous_gqa_decode",
    "varlen_gqa_decode_with_sink_logits": "intent_hip_varlen_decode_sink",
    "splitk_attention_f32_to_f16_reduce": "intent_hip_splitk_reduce_f32_to_f16",
    "csr_spmm": "intent_hip_csr_spmm_f32", "csr_spmv": "intent_hip_csr_spmv_f32",
    "qk_norm_rope_f16": "intent_hip_qk_norm_rope", "qk_norm_rope_bf16": "intent_hip_qk_norm_rope",
    "qk_norm_rope_backward_f16": "intent_hip_qk_norm_rope_backward",
    "qk_norm_rope_backward_bf16": "intent_hip_qk_norm_rope_backward",
    "paged_cache_append_f16": "intent_hip_paged_cache_append", "paged_cache_append_bf16": "intent_hip_paged_cache_append",
    "paged_cache_read_f16": "intent_hip_paged_cache_read", "paged_cache_read_bf16": "intent_hip_paged_cache_read",
    "paged_gqa_decode_mx_f16": "intent_hip_paged_gqa_decode_mx", "paged_gqa_decode_mx_bf16": "intent_hip_paged_gqa_decode_mx",
    "linear_mxfp4_f16": "intent_hip_linear_mxfp4", "linear_mxfp4_bf16": "intent_hip_linear_mxfp4",
    **{f"{name}_{element}": "intent_hip_" + name for element in ("f16", "bf16")
       for name in ("residual_norm", "residual_norm_i8", "residual_norm_backward", "quantize_rows", "swiglu_quantize_rows", "linear_i8",
                    "paged_gqa_decode_prefix")},
}
assert set(ENTRY_POINTS) == set(SPECS)


def signature_of(interface) -> tuple:
    from ..interface import ViewParameter

    return tuple(("view", int(p.access), p.dtype.name, p.rank) if isinstance(p, ViewParameter)
                 else ("scalar", p.dtype.name) for p in interface.parameters)


def recognize(definition, interface, constexpr_names: tuple[str, ...]) -> OperatorSpec:
    name = getattr(definition, "__name__", None)
    spec = SPECS.get(name)
    if spec is None:
        raise CompilationStageError(
            "provider_recognition", f"the hip provider has no kernel for definition {name!r}; "
            f"supported: {', '.join(sorted(SPECS))}")
    if signature_of(interface) != spec.signature or tuple(constexpr_names) != spec.constexprs:
        raise CompilationStageError(
            "provider_recognition", f"definition {name!r} does not have the signature the hip kernel implements: "
            f"expected {spec.signature} with constexprs {spec.constexprs}, got {signature_of(interface)} "
            f"with constexprs {tuple(constexpr_names)}")
    return spec


def recognize_saved(name: str, signature: tuple, constexpr_names: tuple[str, ...]) -> OperatorSpec:
    """Recognition of a saved program (no definition object): by name, signature and constexprs."""
    spec = SPECS.get(name)
    if spec is None or tuple(signature) != spec.signature or tuple(constexpr_names) != spec.constexprs:
        raise CompilationStageError("provider_recognition",
                                    f"saved program {name!r} does not match a kernel of this hip provider")
    return spec
