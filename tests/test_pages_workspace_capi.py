"""The page operators' workspace through the C-ABI: a buffer smaller than qwa_kv_pages_work_bytes is refused before anything is
launched (addresses below are never dereferenced)."""
import ctypes

import pytest

import qwengine_amd.ops as ops
from test_pages_capi import P, FakePages, layer

# (requests and tables for which each operator's own part of the buffer is the largest)
TABLES = {"extend": FakePages(n_seq=4, ld=8, n_pages=16), "fork": FakePages(n_seq=1024, ld=500, n_pages=16),
          "compact": FakePages(n_seq=4, ld=8, n_pages=40000)}


def call(which, pages, size):
    L, pc, arr = ops.lib(), ctypes.byref(pages.c()), ctypes.byref(layer(cap=40000 * 64).c())
    if which == "extend":
        return L.qwa_kv_pages_extend(pc, P, P, 2, arr, 1, ops.Q8_0, P, P, size, None)
    if which == "fork":
        return L.qwa_kv_pages_fork(pc, P, P, 2, P, size, None)
    return L.qwa_kv_pages_compact(pc, arr, 1, ops.Q8_0, P, P, size, None)


@pytest.mark.parametrize("tables", TABLES)
@pytest.mark.parametrize("which", ["extend", "fork", "compact"])
def test_small_workspaces_are_refused(which, tables):
    pages = TABLES[tables]
    need = ops.kv_pages_work_bytes(pages)
    assert need > 0
    for size in (0, 1, need // 2, need - 1):
        assert call(which, pages, size) == 2  # QWA_ERR_RANGE
        assert f"workspace of {size} bytes, the call needs {need}" in ops.lib().qwa_last_error().decode()
