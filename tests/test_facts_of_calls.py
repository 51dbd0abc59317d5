"""What the entry points say on the host about a call agrees with what the call itself asks for; nothing is launched."""
import ctypes
import re

import pytest

from intent_amd.runtime.hip import library as hiplib


@pytest.mark.parametrize("pages,ps", [(0, 64), (0, 16), (0, 0), (9, 0), (9, 64)])
@pytest.mark.parametrize("batch,positions", [(4, 50001), (2, 4000), (64, 8193)])
def test_decode_workspace_of_any_cache(pages, ps, batch, positions):
    """A cache without a page or a token is cut as its query says, however long the table."""
    lib, size = hiplib.library(), ctypes.c_size_t(0)
    assert lib.fn["paged_gqa_decode_mx_workspace_bytes"](batch, 32, 8, 4, 128, ps, positions, ctypes.byref(size)) == 0
    assert size.value > 0
    strides = (ctypes.c_int64 * 22)(4096, 128, 1, *(65536, 1024, 128, 1, 2048, 32, 4, 1) * 2, 4096, 128, 1)
    assert lib.fn["paged_gqa_decode_mx"](hiplib.F16, *[256] * 9, batch, 32, 8, 4, 128, pages, ps, positions, strides, 0.1, 256,
                                         size.value - 1, None) == 5
    assert int(re.search(rb"needs (\d+) workspace", lib.fn["last_error"]()).group(1)) == size.value


def test_norm_rope_of_too_many_heads():
    """Numbers of heads whose walk would leave 32 bits are refused before any launch, and by the query."""
    lib, size = hiplib.library(), ctypes.c_size_t(0)
    strides = (ctypes.c_int64 * 22)(*(2 ** 34, 16, 1) * 2, 8, 1, 8, 1, *(2 ** 34, 16, 1) * 4)
    for q_heads, kv_heads in ((2 ** 30 - 1, 2 ** 30 - 1), (2 ** 30 - 1, 1), (1, 2 ** 30 - 1)):
        assert lib.fn["qk_norm_rope"](hiplib.F16, *[256] * 9, 2, q_heads, kv_heads, 16, 9, 8, strides, 0.0, 0, None) == 2
        assert b"too large" in lib.fn["last_error"]()
        assert lib.fn["qk_norm_rope_backward"](hiplib.F16, *[256] * 13, 2, q_heads, kv_heads, 16, 9, 8, strides, 0.0, 0, 256, 2 ** 40,
                                               None) == 2
        assert lib.fn["qk_norm_rope_backward_workspace_bytes"](2, q_heads, kv_heads, 16, ctypes.byref(size)) == 2
    assert lib.fn["qk_norm_rope_backward_workspace_bytes"](2, 2 ** 29 - 1, 2 ** 29 - 1, 16, ctypes.byref(size)) == 0
