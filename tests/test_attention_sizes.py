"""Sizes of pace_kv_attention and its workspace, found on the host (no GPU)."""
import ctypes

import pytest

from paceserve_amd import _native

LIB = _native.load()
EINVAL, ERANGE = _native.PACE_KV_EINVAL, _native.PACE_KV_ERANGE


def workspace(batch=1, heads=8, group=4, D=128, max_q=1, num_indices=8192, page=16):
    out = ctypes.c_int64(-1)
    return LIB.pace_kv_attention_workspace(batch, heads, group, D, max_q, num_indices, page, ctypes.byref(out)), out.value


@pytest.mark.parametrize("sizes", [
    # (requests + 8) * heads * row tiles = 2^10 * 2^30 * 2^24 = 2^64
    dict(batch=1016, heads=1 << 30, group=1, D=256, max_q=(1 << 30) - 1, num_indices=0),
    # 2^20 * 2^20 * 2^24
    dict(batch=(1 << 20) - 8, heads=1 << 20, group=1, D=256, max_q=(1 << 30) - 1, num_indices=0),
    # pages * heads * row tiles past 2^63
    dict(heads=1 << 30, group=1, D=256, max_q=(1 << 30) - 1, num_indices=1 << 26),
    # tokens past 2^63
    dict(num_indices=1 << 60, page=16), dict(num_indices=(1 << 62) + 1, page=4),
    dict(batch=1 << 24, heads=1, num_indices=0), dict(batch=(1 << 31) - 1, num_indices=0)])
def test_products_past_64_bits_are_refused(sizes):
    assert workspace(**sizes)[0] == ERANGE
    assert "too many" in LIB.pace_kv_last_error().decode() or "more than" in LIB.pace_kv_last_error().decode()


def test_a_call_of_such_sizes_is_refused():
    assert LIB.pace_kv_attention(0x1000, 1 << 30, 0, 1, 0x100, (1 << 20) - 8, 1 << 20, 1, 256, 0x2000, 0, 1, 1, 0x100, 0,
                                 0x100, 0x100, (1 << 30) - 1, None, 0, 0.1, 0.0, 0x3000, 1 << 30, None, None, 0, None,
                                 None) == ERANGE


@pytest.mark.parametrize("batch,num_indices,max_q", [(256, 33024, 512), (256, 33024, 1024), (1024, 132096, 512)])
def test_requests_that_are_not_split_take_no_workspace(batch, num_indices, max_q):
    """One long draft beside many single tokens: only requests longer than a chunk have
    parts, and all of them together at most twice as many as whole chunks fit the pages."""
    rc, size = workspace(batch=batch, heads=8, group=8, max_q=max_q, num_indices=num_indices)
    rows = 8 * max_q * 8                                   # of all heads
    # rows enough to fill the CUs: chunks of a third of all pages, or more
    assert rc == 0 and size <= 2 * 3 * rows * (128 + 2) * 4


def test_a_pool_without_pages_needs_no_memory():
    def call(pages, space):
        return LIB.pace_kv_attention(0x1000, 8192, 0, 8, 0x100, 2, 8, 4, 128, None, 0, pages, 16, 0x100, 4096, 0x100,
                                     0x100, 4, None, 0, 0.1, 0.0, 0x3000, 8192, None, space, 0, None, None)

    assert call(9, None) == EINVAL and "NULL" in LIB.pace_kv_last_error().decode()
    assert call(0, None) == EINVAL and "workspace" in LIB.pace_kv_last_error().decode()  # the next thing it lacks
