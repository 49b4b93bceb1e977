"""Sizes of pace_kv_attention and its workspace, found on the host (no GPU)."""
import ctypes

import pytest

from paceserve_amd import _native

LIB = _native.load()


def workspace(batch=1, heads=8, group=4, D=128, max_q=1, num_indices=8192, page=16):
    out = ctypes.c_int64(-1)
    return LIB.pace_kv_attention_workspace(batch, heads, group, D, max_q, num_indices, page, ctypes.byref(out)), out.value


@pytest.mark.parametrize("batch,num_indices,max_q", [(256, 33024, 512), (256, 33024, 1024), (1024, 132096, 512)])
def test_requests_that_are_not_split_take_no_workspace(batch, num_indices, max_q):
    """One long draft beside many single tokens: only requests longer than a chunk have
    parts, and all of them together at most twice as many as whole chunks fit the pages."""
    rc, size = workspace(batch=batch, heads=8, group=8, max_q=max_q, num_indices=num_indices)
    rows = 8 * max_q * 8                                   # of all heads
    # rows enough to fill the CUs: chunks of a third of all pages, or more
    assert rc == 0 and size <= 2 * 3 * rows * (128 + 2) * 4
