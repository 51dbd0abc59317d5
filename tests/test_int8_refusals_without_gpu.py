"""The entry points of the norm of the stream, of 8-bit rows and products and of the decode behind a prefix refuse bad requests on the
host, before any HIP call; empty work is a successful no-op."""
import ctypes

import pytest

from intent_amd.runtime.hip import library as hiplib
from intent_amd.runtime.hip.operators import SPECS

F16, BF16 = hiplib.F16, hiplib.BF16


def strides(*values):
    return (ctypes.c_int64 * len(values))(*values)


@pytest.mark.parametrize("narrow", [False, True])
def test_residual_norm(narrow):
    lib = hiplib.library()
    err = lambda: lib.fn["last_error"]()  # noqa: E731

    def call(dtype=F16, block=16, gate=16, post=16, weight=16, out=16, scales=16, tokens=4, d=64, gates=4, posts=64,
             of=(64, 64, 1, 64, 64)):
        outputs = (out, scales) if narrow else (out,)
        return lib.fn["residual_norm_i8" if narrow else "residual_norm"](
            dtype, block, 16, gate, post, weight, 16, *outputs, tokens, d, gates, posts, strides(*of), 1.0, 1.0, 1e-6, None)

    assert call(dtype=hiplib.F32) == 1 and b"F16 or BF16" in err()
    assert call(tokens=-1) == 1 and call(gates=-1) == 1 and b"negative" in err()
    assert call(gates=3) == 1 and b"gates" in err()
    assert call(posts=32) == 1 and b"weights" in err()
    assert call(d=16385, posts=0) == 2 and b"16384" in err()
    assert call(tokens=2 ** 40, gates=0) == 2 and call(tokens=2 ** 31 - 1, gates=0) == 2 and b"too large" in err()
    assert call(block=None) == 1 and call(gate=None) == 1 and call(post=None) == 1 and call(weight=None) == 1 and call(out=None) == 1
    assert b"null" in err()
    assert call(of=(64, -64, 1, 64, 64)) == 1 and b"negative stride" in err()
    assert call(tokens=0, gates=0, block=None) == 0
    if narrow:
        assert call(scales=None) == 1
    else:
        assert call(d=0, posts=0, block=None) == 0


def test_residual_norm_backward():
    lib = hiplib.library()
    err = lambda: lib.fn["last_error"]()  # noqa: E731
    size = ctypes.c_size_t(0)
    query = lib.fn["residual_norm_backward_workspace_bytes"]

    def call(dtype=F16, block=16, grad=16, gate=16, grad_gate=16, grad_post=16, grad_weight=16, tokens=4, d=64, gates=4, posts=64,
             of=(64, 64, 1, 64, 64, 64, 64, 1), workspace=None, size=0):
        return lib.fn["residual_norm_backward"](dtype, block, 16, gate, 16, 16, grad, 16, 16, 16, grad_gate, grad_post, grad_weight, tokens, d,
                                                gates, posts, strides(*of), 1.0, 1.0, 1e-6, workspace, size, None)

    assert call(dtype=9) == 1 and call(gates=2) == 1 and call(posts=2) == 1 and call(d=2 ** 20, posts=0) == 2
    assert call(grad_weight=None) == 1 and call(grad_post=None) == 1 and call(grad_gate=None) == 1 and b"null" in err()
    assert call(block=None) == 1 and call(grad=None) == 1
    assert call(of=(64, 64, 1, 64, 64, -64, 64, 1)) == 1
    assert call() == 5 and b"workspace" in err()
    assert query(4, 64, 64, ctypes.byref(size)) == 0 and 2 * 64 * 4 <= size.value <= 4 * 2 * 64 * 4
    assert call(workspace=256, size=size.value - 1) == 5 and call(workspace=264, size=size.value) == 5
    assert query(16384, 4096, 0, ctypes.byref(size)) == 0 and 0 < size.value <= 4096 * 4096 * 4
    assert query(0, 64, 64, ctypes.byref(size)) == 0 and size.value == 0
    assert query(4, 64, 64, None) == 1 and query(4, 64, 3, ctypes.byref(size)) == 1


def test_quantize_rows():
    lib = hiplib.library()
    err = lambda: lib.fn["last_error"]()  # noqa: E731

    def plain(dtype=F16, x=16, out=16, scales=16, rows=4, d=64, ldx=64, ldo=64):
        return lib.fn["quantize_rows"](dtype, x, out, scales, rows, d, ldx, ldo, None)

    def gated(dtype=F16, up=16, out=16, scales=16, rows=4, d=64, ldu=64, **rest):
        return lib.fn["swiglu_quantize_rows"](dtype, 16, up, out, scales, rows, d, 64, ldu, 64, None)

    for call in (plain, gated):
        assert call(dtype=hiplib.F32) == 1 and b"F16 or BF16" in err()
        assert call(rows=-1) == 1 and call(d=-1) == 1 and b"negative" in err()
        assert call(d=32769) == 2 and b"32768" in err()
        assert call(rows=2 ** 40) == 2
        assert call(out=None) == 1 and call(scales=None) == 1 and b"null" in err()
        assert call(rows=0, out=None) == 0
    assert plain(x=None) == 1 and gated(up=None) == 1
    assert plain(ldx=-1) == 1 and gated(ldu=-1) == 1 and b"negative stride" in err()


def test_linear_i8():
    lib = hiplib.library()
    err = lambda: lib.fn["last_error"]()  # noqa: E731

    def call(dtype=F16, x=16, w=16, xs=16, ws=16, bias=None, y=16, m=4, n=8, k=64, ldx=64, ldw=64, ldy=8, workspace=None, size=0):
        return lib.fn["linear_i8"](dtype, x, w, xs, ws, bias, y, m, n, k, ldx, ldw, ldy, workspace, size, None)

    assert call(dtype=hiplib.F32) == 1 and b"F16 or BF16" in err()
    assert call(m=-1) == 1 and call(ldw=-64) == 1 and b"negative" in err()
    assert call(k=40) == 2 and b"multiples of 16" in err()
    assert call(k=131072) == 2 and b"131072" in err()
    assert call(x=None) == 1 and call(w=None) == 1 and call(xs=None) == 1 and call(ws=None) == 1 and call(y=None) == 1 and b"null" in err()
    assert call(x=24) == 2 and call(ldx=65) == 2 and b"aligned" in err()
    assert call(w=24) == 2 and call(ldw=72) == 2 and b"weight rows" in err()
    assert call(y=17) == 1
    assert call(m=2 ** 21) == 2 and call(n=2 ** 30) == 2 and call(m=2 ** 20, n=2 ** 22) == 2
    assert call(m=0, x=None) == 0 and call(n=0) == 0
    size = ctypes.c_size_t(0)
    query = lib.fn["linear_i8_workspace_bytes"]
    assert query(1, 14336, 4096, ctypes.byref(size)) == 0 and size.value == 0
    assert query(100, 64, 4096, ctypes.byref(size)) == 0 and size.value % (100 * 64 * 4) == 0 and size.value > 0
    assert call(m=100, n=64, k=4096, ldx=4096, ldw=4096, ldy=64) == 5 and b"workspace" in err()
    assert call(m=100, n=64, k=4096, ldx=4096, ldw=4096, ldy=64, workspace=256, size=size.value - 1) == 5
    assert query(4, 8, 40, ctypes.byref(size)) == 2 and query(4, 8, 64, None) == 1


def test_prefix_decode():
    lib = hiplib.library()
    err = lambda: lib.fn["last_error"]()  # noqa: E731
    rows, cache = (4096, 128, 1), (65536, 1024, 128, 1)
    size = ctypes.c_size_t(0)
    query = lib.fn["paged_gqa_decode_prefix_workspace_bytes"]

    def call(dtype=F16, q=16, keys=16, shared=16, length=16, own=16, out=16, b=2, heads=32, kv=8, group=4, d=128, pages=9, ps=64, prefix=4,
             positions=4, groups=(rows, cache, cache, rows), workspace=None, size=0):
        return lib.fn["paged_gqa_decode_prefix"](dtype, q, keys, 16, shared, length, 16, own, 16, out, b, heads, kv, group, d, pages, ps, prefix,
                                                 positions, strides(*(s for g in groups for s in g)), 0.1, workspace, size, None)

    assert call(dtype=hiplib.F32) == 1 and b"F16 or BF16" in err()
    assert call(b=-1) == 1 and call(prefix=-1) == 1 and b"negative" in err()
    assert call(group=3) == 1 and call(group=0) == 1 and b"HEAD_GROUP" in err()
    assert call(d=96) == 2 and b"64 or 128" in err()
    assert call(q=None) == 1 and call(keys=None) == 1 and call(shared=None) == 1 and call(length=None) == 1 and call(own=None) == 1
    assert call(out=None) == 1 and b"null" in err()
    assert call(q=18) == 2 and call(keys=24) == 2 and b"aligned" in err()
    assert call(groups=(rows, (65536, 1024, 132, 1), cache, rows)) == 2
    assert call(groups=(rows, cache, cache, (4096, 128, 2))) == 1 and b"unit inner" in err()
    assert call(groups=((-4096, 128, 1), cache, cache, rows)) == 1 and b"negative stride" in err()
    assert call(b=2 ** 30) == 2 and call(prefix=2 ** 27, ps=64) == 2 and call(positions=2 ** 30) == 2 and b"too large" in err()
    assert call(b=0) == 0 and call(heads=0, kv=0) == 0
    assert query(2, 32, 8, 4, 128, 64, 4, 4, ctypes.byref(size)) == 0 and size.value > 0
    assert call(size=size.value) == 5 and call(workspace=256, size=size.value - 1) == 5 and b"workspace" in err()
    assert query(2, 32, 8, 4, 128, 64, 4, 4, None) == 1 and query(2, 32, 8, 3, 128, 64, 4, 4, ctypes.byref(size)) == 1
    # the last part of a prefix ends within 31 bits; pages without tokens have no jobs
    assert call(prefix=2 ** 25 - 2 ** 13, ps=64) == 2 and b"too large" in err()
    assert query(1, 1, 1, 1, 64, 0, 0, 2 ** 28, ctypes.byref(size)) == 0 and size.value <= 2 * 66 * 4
    # blocks and states are counted in 32 bits whatever the tables hold
    for b, kv, group, ps, prefix, positions in ((2 ** 20, 1, 1, 1, 2 ** 28, 2 ** 28), (1, 1, 1, 2 ** 12, 0, 2 ** 28), (64, 8, 8, 16, 2 ** 20, 2 ** 20)):
        assert query(b, kv * group, kv, group, 64, ps, prefix, positions, ctypes.byref(size)) == 0
        assert size.value // (66 * 4) <= 2 ** 31


def test_facts_of_calls():
    """The resource entry points take any sizes: an answer (where there is a GPU) or an error, never the end of the process."""
    lib = hiplib.library()
    for op in range(hiplib.OP_RESIDUAL_NORM, hiplib.OP_PAGED_GQA_DECODE_PREFIX + 1):
        for rows in (-1, 0, 1, 7, 2 ** 40):
            for cols in (-1, 0, 1, 128, 2 ** 40):
                lib.kernel_resources(op, F16, rows, cols)
        for count in (0, 2, 3, 7, 9):
            for value in (-1, 0, 1, 128, 2 ** 40):
                lib.call_resources(op, BF16, *[value] * count)


def test_rows_that_may_be_one():
    """Which views of the norm may be one: rows with rows, never a token's numbers with a column's."""
    norm, narrow, back = (SPECS[n + "bf16"] for n in ("residual_norm_", "residual_norm_i8_", "residual_norm_backward_"))
    assert norm.may_be_one(1, 5) and norm.may_be_one(0, 6) and not norm.may_be_one(4, 5) and not norm.may_be_one(5, 6)
    assert narrow.may_be_one(1, 5) and not narrow.may_be_one(0, 6) and not narrow.may_be_one(4, 7)
    assert back.may_be_one(5, 7) and back.may_be_one(1, 8) and not back.may_be_one(4, 9) and not back.may_be_one(2, 9)
    assert SPECS["stable_softmax"].may_be_one(0, 1) and not SPECS["linear_i8_f16"].may_be_one(0, 5)
