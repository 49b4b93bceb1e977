"""Argument errors of pace_kv_attention that the library finds on the host, and
the oracle against torch's softmax (no GPU)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import attention_oracle as ao
from paceserve_amd import _native

LIB = _native.load()
EINVAL, ERANGE = _native.PACE_KV_EINVAL, _native.PACE_KV_ERANGE


def call(q=0x1000, stride=8192, type=0, nnz=8, qo=0x100, batch=2, heads=8, group=4, D=128, cache=0x2000, fmt=0,
         pages=9, P=16, indices=0x100, num_indices=6, indptr=0x100, last=0x100, max_q=4, mask=None, words=0, scale=0.1,
         cap=0.0, out=0x3000, out_stride=8192, space=None, size=0):
    return LIB.pace_kv_attention(q, stride, type, nnz, qo, batch, heads, group, D, cache, fmt, pages, P, indices,
                                 num_indices, indptr, last, max_q, mask, words, scale, cap, out, out_stride, None,
                                 space, size, None, None)


@pytest.mark.parametrize("args,code,msg", [
    (dict(nnz=-1), EINVAL, "negative"), (dict(batch=-1), EINVAL, "positive"), (dict(heads=0), EINVAL, "positive"),
    (dict(group=0), EINVAL, "positive"), (dict(max_q=0), EINVAL, "positive"), (dict(P=0), EINVAL, "positive"),
    (dict(D=96), EINVAL, "head_dim"), (dict(type=2), EINVAL, "bfloat16 or float16"), (dict(fmt=3), EINVAL, "format"),
    (dict(pages=-1), ERANGE, "pages"), (dict(pages=1 << 31), ERANGE, "pages"), (dict(cap=-1.0), EINVAL, "soft_cap"),
    (dict(cap=math.nan), EINVAL, "soft_cap"), (dict(cap=math.inf), EINVAL, "soft_cap"),
    (dict(scale=math.nan), EINVAL, "scale"), (dict(q=None), EINVAL, "NULL"), (dict(out=None), EINVAL, "NULL"),
    (dict(cache=None), EINVAL, "NULL"), (dict(indices=None), EINVAL, "NULL"), (dict(indptr=None), EINVAL, "NULL"),
    (dict(last=None), EINVAL, "NULL"), (dict(qo=None), EINVAL, "one token"),
    (dict(mask=0x100, words=0), EINVAL, "mask"), (dict(mask=0x100, words=1, max_q=65), EINVAL, "mask"),
    (dict(mask=0x104, words=1), EINVAL, "aligned"), (dict(stride=8184), EINVAL, "strides"),
    (dict(stride=8200), EINVAL, "strides"), (dict(out_stride=8188), EINVAL, "strides"),
    (dict(q=0x1008), EINVAL, "aligned"), (dict(cache=0x2008), EINVAL, "aligned"), (dict(out=0x3004), EINVAL, "aligned"),
    (dict(pages=1 << 21, P=16), ERANGE, "64 GiB"), (dict(num_indices=1 << 27), ERANGE, "tokens"),
    (dict(nnz=1 << 20, max_q=1 << 20, stride=8192), ERANGE, "query rows"),
    (dict(fmt=1, heads=1, P=1, D=64, stride=512, out_stride=512), EINVAL, "multiple of 16"),
    (dict(num_indices=4096), EINVAL, "workspace"), (dict(num_indices=4096, space=0x1000, size=64), EINVAL, "workspace"),
    (dict(num_indices=4096, space=0x1008, size=1 << 40), EINVAL, "workspace")])
def test_refuses(args, code, msg):
    assert call(**args) == code
    assert msg in LIB.pace_kv_last_error().decode()


def test_nothing_to_do():
    assert call(nnz=0) == 0 and call(batch=0) == 0


def test_workspace_size():
    out = ctypes.c_int64()
    assert LIB.pace_kv_attention_workspace(2, 8, 4, 128, 4, 4, 16, ctypes.byref(out)) == 0 and out.value == 0
    assert LIB.pace_kv_attention_workspace(1, 8, 4, 128, 1, 8192, 16, ctypes.byref(out)) == 0 and out.value > 0
    assert LIB.pace_kv_attention_workspace(1, 8, 4, 128, 1, 8192, 16, None) == EINVAL
    assert LIB.pace_kv_attention_workspace(1, 8, 4, 100, 1, 8192, 16, ctypes.byref(out)) == EINVAL


def test_scales_past_float32_are_refused():
    assert call(scale=math.inf) == EINVAL and call(scale=math.nan) == EINVAL
    assert call(cap=1e-44) == EINVAL and "soft_cap" in LIB.pace_kv_last_error().decode()   # scale / soft_cap


def test_sizes_whose_products_pass_32_bits():
    """3 * 2^27 pages times 2^13 heads, a request of which is never cut: no parts are kept."""
    out = ctypes.c_int64(-1)
    assert LIB.pace_kv_attention_workspace(1, 1 << 13, 1, 128, 1, 3 << 27, 1, ctypes.byref(out)) == 0 and out.value == 0


def test_oracle_against_torch():
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((3, 4, 64)), rng.standard_normal((20, 2, 64)), rng.standard_normal((20, 2, 64))
    mask = np.array([[1], [3], [5]], np.uint64)
    sees = ao.visible(20, 3, mask)
    assert sees[:, :17].all() and sees[:, 17:].tolist() == [[True, False, False], [True, True, False],
                                                            [True, False, True]]
    out, lse, *_ = ao.attend(q, k, v, 0.125, 30.0, sees)
    tq = torch.from_numpy(q).transpose(0, 1)
    tk, tv = (torch.from_numpy(np.repeat(x, 2, 1)).transpose(0, 1) for x in (k, v))
    s = 30 * torch.tanh(tq @ tk.transpose(1, 2) * 0.125 / 30)
    s = s.masked_fill(~torch.from_numpy(sees), -math.inf)
    assert np.allclose(out, (torch.softmax(s, -1) @ tv).transpose(0, 1).numpy(), atol=1e-12)
    assert np.allclose(lse, torch.logsumexp(s, -1).T.numpy(), atol=1e-12)
