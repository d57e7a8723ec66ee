"""Tiles too large for one launch of the paged cache's moves are refused (no GPU: nothing is launched)."""
import ctypes

import pytest

from nntile_amd import hip_sdpa as h


@pytest.mark.parametrize("t,head,rows", [("fp32", 128, 1 << 28), ("fp32", 64, 1 << 28), ("bf16", 128, 1 << 28),
                                         ("fp16", 64, 1 << 28)])
def test_tiles_of_128_gib(t, head, rows):
    """2^30 rows of 128 bytes and more take 2^32 threads and more: a launch would run a part of them."""
    L = h.lib()
    c = h.PagedCacheArgs()
    c.k_pages = c.v_pages = c.table = c.lens = 4096         # never dereferenced on these paths
    c.head, c.page_rows, c.n_head_kv, c.n_pages, c.max_pages, c.n_batch = head, 1024, 2, 5, 1 << 20, 2
    c.page_stride = head * 1024 * 2
    assert getattr(L, "nntile_hip_paged_kv_append_" + t)(None, ctypes.byref(c), rows, 4096, 4096) == h.EINVAL
    assert getattr(L, "nntile_hip_paged_kv_read_" + t)(None, ctypes.byref(c), 0, rows, 4096, 4096) == h.EINVAL
