"""Refusals of the page operations that come before anything is launched, and so before any state has changed."""
import ctypes

import pytest

from vllm_xpu_kernels import cabi

INVALID, TOO_LARGE = 1, 4


@pytest.fixture()
def buf():
    b = (ctypes.c_char * 8192)()
    return (ctypes.addressof(b) + 63) // 64 * 64, b  # a 64-byte aligned address, and what keeps it alive


@pytest.mark.parametrize("rows,row_bytes", [(1 << 31, 2), (1 << 30, 64), (1, 1 << 45), (1 << 62, 1 << 20), (1, (1 << 63) - 1)])
def test_pages_that_fit_no_launch(buf, rows, row_bytes):
    """fork and compact change lengths, counts and tables in a launch of their own: a page too large for the copies that follow
    is refused before it, by the same answer as copy_blocks gives."""
    L, p = cabi.lib(), buf[0]
    caches = (ctypes.c_void_p * 2)(p, p)
    geometry = (512, rows, row_bytes, 512)
    assert L.kvc_copy_blocks(caches, 2, p, 1, 64, *geometry, None) == TOO_LARGE
    assert L.kvc_copy_blocks(caches, 2, p, 0, 64, *geometry, None) == 0
    assert L.kvc_fork_blocks(p, p, p, p, p, 2, 4, 8, 8, 64, 16, caches, 2, *geometry, p, p, None) == TOO_LARGE
    assert "fork_blocks: a page is too large" in cabi.last_error()
    assert L.kvc_compact_blocks(p, p, 4, 8, 8, 64, caches, 2, *geometry, p, 4, None) == TOO_LARGE
    assert "compact_blocks: a page is too large" in cabi.last_error()


def test_more_rows_than_a_launch_has_ctas(buf):
    L, p = cabi.lib(), buf[0]
    caches = (ctypes.c_void_p * 2)(p, p)
    assert L.kvc_compact_blocks(p, p, 0x7FFFFFFF, 8, 8, 64, caches, 2, 512, 1, 512, 512, p, 4, None) == INVALID
