"""The entry points without a reference counterpart refuse bad requests on the host, before any HIP call; empty work is a
successful no-op."""
import ctypes

from intent_amd.runtime.hip import library as hiplib

F16, BF16 = hiplib.F16, hiplib.BF16


def strides(*groups):
    values = [s for group in groups for s in group]
    return (ctypes.c_int64 * len(values))(*values)


def test_norm_rope():
    lib = hiplib.library()
    err = lambda: lib.fn["last_error"]()  # noqa: E731
    good = [(1024, 128, 1), (1024, 128, 1), (64, 1), (64, 1), (1024, 128, 1), (1024, 128, 1)]

    def call(dtype=F16, q=16, positions=16, tokens=4, heads=8, kv=2, d=128, table=100, pairs=64, groups=good):
        return lib.fn["qk_norm_rope"](dtype, q, 16, 16, 16, positions, 16, 16, 16, 16, tokens, heads, kv, d, table, pairs,
                                      strides(*groups), 1e-6, 0, None)

    assert call(dtype=hiplib.F32) == 1 and b"dtype" in err()
    assert call(tokens=-1) == 1 and b"negative" in err()
    assert call(pairs=65) == 1 and b"do not fit" in err()
    assert call(d=1025) == 2 and b"1024" in err()
    assert call(q=None) == 1 and b"null" in err()
    assert call(positions=None) == 1 and b"null" in err()
    assert call(table=0) == 1 and b"hold no position" in err()
    assert call(groups=[(1024, 128, 2)] + good[1:]) == 1 and b"unit inner stride" in err()
    assert call(groups=[(-1024, 128, 1)] + good[1:]) == 1 and b"negative stride" in err()
    assert call(groups=good[:2] + [(64, 2)] + good[3:]) == 1 and b"tables" in err()
    assert call(tokens=2 ** 40) == 2
    assert call(tokens=0, q=None) == 0 and call(d=0, pairs=0) == 0 and call(heads=0, kv=0) == 0

    size = ctypes.c_size_t(0)
    query = lib.fn["qk_norm_rope_backward_workspace_bytes"]
    assert query(16384, 32, 8, 128, ctypes.byref(size)) == 0 and 0 < size.value <= 4096 * 2 * 128 * 4
    assert query(0, 32, 8, 128, ctypes.byref(size)) == 0 and size.value == 0
    assert query(16384, 32, 8, 128, None) == 1 and query(-1, 32, 8, 128, ctypes.byref(size)) == 1
    assert query(4, 32, 8, 128, ctypes.byref(size)) == 0
    rows = [(1024, 128, 1)] * 4

    def back(workspace=256, bytes_=size.value, grad=16, weight=16, tokens=4, d=128):
        return lib.fn["qk_norm_rope_backward"](BF16, 16, 16, 16, 16, 16, 16, 16, grad, 16, 16, 16, weight, 16, tokens, 8, 2, d,
                                               100, 32, strides(*good[:4], *rows), 1e-6, 1, workspace, bytes_, None)

    assert back(workspace=None) == 5 and b"workspace" in err()
    assert back(bytes_=16) == 5 and back(workspace=264) == 5
    assert back(grad=None) == 1 and back(weight=None) == 1 and back(d=2000) == 2


def test_paged_cache():
    lib = hiplib.library()
    err = lambda: lib.fn["last_error"]()  # noqa: E731
    rows, held, powers = (1024, 128, 1), (65536, 1024, 128, 1), (2048, 32, 4, 1)

    def call(reading=False, dtype=F16, k=16, keys=16, cu=16, n=4, b=2, heads=8, d=128, dv=128, pages=9, ps=64, positions=4,
             groups=(rows, rows, held, powers, held, powers), lengths=16):
        tail = (n, b, heads, d, dv, pages, ps, positions, strides(*groups), None)
        if reading:
            return lib.fn["paged_cache_read"](dtype, keys, 16, 16, 16, cu, 16, 16, k, 16, *tail)
        return lib.fn["paged_cache_append"](dtype, k, 16, keys, 16, 16, 16, cu, 16, 16, lengths, *tail)

    for reading in (False, True):
        assert call(reading, dtype=hiplib.F32) == 1 and b"F16 or BF16" in err()
        assert call(reading, n=-1) == 1 and b"negative" in err()
        assert call(reading, d=48) == 2 and b"blocks of 32" in err()
        assert call(reading, k=None) == 1 and call(reading, keys=None) == 1 and call(reading, cu=None) == 1
        assert call(reading, k=18) == 2 and b"aligned" in err()
        assert call(reading, keys=24) == 2 and b"aligned" in err()
        assert call(reading, ps=0) == 1 and b"no token" in err()
        assert call(reading, groups=((1028, 128, 1), rows, held, powers, held, powers)) == 2
        assert call(reading, groups=(rows, rows, (65536, 1024, 136, 1), powers, held, powers)) == 2
        assert call(reading, groups=(rows, rows, held, (2048, 32, 4, 2), held, powers)) == 1 and b"unit inner" in err()
        assert call(reading, groups=(rows, (-1024, 128, 1), held, powers, held, powers)) == 1
        assert call(reading, heads=2 ** 28) == 2 and call(reading, n=2 ** 40) == 2
        assert call(reading, n=0) == 0 and call(reading, b=0) == 0 and call(reading, heads=0) == 0
    assert call(lengths=None) == 1
    assert call(pages=0) == 0 and call(positions=0) == 0            # nowhere to write


def test_decode_mx():
    lib = hiplib.library()
    err = lambda: lib.fn["last_error"]()  # noqa: E731
    rows, held, powers = (4096, 128, 1), (65536, 1024, 128, 1), (2048, 32, 4, 1)

    def call(dtype=F16, q=16, keys=16, out=16, b=2, heads=32, kv=8, group=4, d=128, pages=9, ps=64, positions=4,
             groups=(rows, held, powers, held, powers, rows), workspace=None, size=0):
        return lib.fn["paged_gqa_decode_mx"](dtype, q, keys, 16, 16, 16, 16, 16, 16, out, b, heads, kv, group, d, pages, ps,
                                             positions, strides(*groups), 0.1, workspace, size, None)

    assert call(dtype=hiplib.F32) == 1 and b"F16 or BF16" in err()
    assert call(b=-1) == 1 and call(group=3) == 1 and b"HEAD_GROUP" in err()
    assert call(d=80) == 2 and b"head widths" in err()
    assert call(q=None) == 1 and call(keys=None) == 1 and call(out=None) == 1
    assert call(q=18) == 2 and call(keys=24) == 2
    assert call(groups=(rows, (65536, 1024, 136, 1), powers, held, powers, rows)) == 2
    assert call(groups=(rows, held, powers, held, powers, (4096, 128, 2))) == 1
    assert call(groups=((-4096, 128, 1), held, powers, held, powers, rows)) == 1
    assert call(b=2 ** 30) == 2 and call(positions=2 ** 30) == 2
    assert call(b=0) == 0 and call(heads=0, kv=0) == 0
    size = ctypes.c_size_t(0)
    query = lib.fn["paged_gqa_decode_mx_workspace_bytes"]
    assert query(2, 32, 8, 4, 128, 64, 4, ctypes.byref(size)) == 0 and size.value == 0       # 256 tokens: a job a sequence
    assert query(8, 32, 8, 4, 128, 64, 1000, ctypes.byref(size)) == 0 and size.value > 0
    assert call(b=8, positions=1000, size=size.value) == 5 and b"workspace" in err()
    assert call(b=8, positions=1000, workspace=256, size=size.value - 1) == 5
    assert query(8, 32, 8, 4, 128, 64, 1000, None) == 1 and query(8, 32, 8, 3, 128, 64, 1000, ctypes.byref(size)) == 1


def test_linear_mxfp4():
    lib = hiplib.library()
    err = lambda: lib.fn["last_error"]()  # noqa: E731

    def call(dtype=F16, x=16, w=16, y=16, m=4, n=8, k=64, ldx=64, ldw=32, lde=2, ldy=8, workspace=None,
             size=0):
        return lib.fn["linear_mxfp4"](dtype, x, w, 16, y, m, n, k, ldx, ldw, lde, ldy, workspace, size, None)

    assert call(dtype=hiplib.F32) == 1 and b"F16 or BF16" in err()
    assert call(m=-1) == 1 and call(ldw=-32) == 1 and b"negative" in err()
    assert call(k=48) == 2 and b"blocks of 32" in err()
    assert call(x=None) == 1 and call(w=None) == 1 and call(y=None) == 1 and b"null" in err()
    assert call(x=24) == 2 and call(ldx=65) == 2 and b"aligned" in err()
    assert call(w=24) == 2 and call(ldw=40) == 2 and b"weight rows" in err()
    assert call(m=2 ** 21) == 2 and call(n=2 ** 30) == 2
    assert call(m=0, x=None) == 0 and call(n=0) == 0
    size = ctypes.c_size_t(0)
    query = lib.fn["linear_mxfp4_workspace_bytes"]
    assert query(1, 14336, 4096, ctypes.byref(size)) == 0 and size.value == 0
    assert query(100, 64, 4096, ctypes.byref(size)) == 0 and size.value % (100 * 64 * 4) == 0 and size.value > 0
    assert call(m=100, n=64, k=4096, ldx=4096, ldw=2048, lde=128, ldy=64) == 5 and b"workspace" in err()
    assert call(m=100, n=64, k=4096, ldx=4096, ldw=2048, lde=128, ldy=64, workspace=256, size=size.value - 1) == 5
    assert query(4, 8, 48, ctypes.byref(size)) == 2 and query(4, 8, 64, None) == 1


def test_facts_of_odd_calls():
    """The resource entry points take any sizes: an answer (where there is a GPU) or an error, never the end of the process."""
    lib = hiplib.library()
    out = hiplib.KernelResources()
    ask = lambda op, *f: lib.fn["call_resources"](op, BF16, (ctypes.c_int64 * len(f))(*f), len(f), ctypes.byref(out))  # noqa: E731
    for op, calls in ((hiplib.OP_PAGED_GQA_DECODE_MX, ((4, 2, 4, 128, 0, 9), (0, 0, 1, 64, 16, 0), (1, 1, 0, 64, 16, 1), (4, 2, 4, 100, 16, 9),
                                                       (-1, 2, 4, 128, 16, 9), (4, 2, 4, 128, 2 ** 40, 2 ** 40), (1, 1, 1, 64, -16, 1))),
                      (hiplib.OP_LINEAR_MXFP4, ((0, 0, 0), (-1, 4, 32), (2 ** 40, 2 ** 40, 32), (1, 1, 33))),
                      (hiplib.OP_QK_NORM_ROPE, ((2 ** 31 - 16, 8, 0, 0), (2 ** 40, 8, 0, 0), (-16, 0, 0, 0), (0, 0, 0, 0), (1025, 0, 0, 1)))):
        for f in calls:
            ask(op, *f)
            assert ask(op, *f[:-1]) == 1
    for f in ((1, 1, 0, 64, 16, 1), (-1, 2, 4, 128, 16, 9), (4, 2, 4, 128, 2 ** 40, 2 ** 40), (1, 1, 1, 64, -16, 1)):
        assert ask(hiplib.OP_PAGED_GQA_DECODE_MX, *f) in (1, 2)
    assert ask(hiplib.OP_QK_NORM_ROPE, 2 ** 31 - 16, 8, 0, 0) == 2 and ask(hiplib.OP_LINEAR_MXFP4, 1, 1, 33) == 2
