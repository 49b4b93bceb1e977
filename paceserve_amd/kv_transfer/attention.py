"""Attention over a paged KV cache on the HIP path: single tokens of a decode
step, or drafted tokens under a tree mask, over a bfloat16 or float16 cache or
a quantised one (mx).

The reader of the pages that the append calls write, with the same tables: in
the reference both belong to one wrapper
(paceserve/model_executor/attention/flashinfer_attention_wrapper.py).
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Tuple, Union

import torch

from .. import _native
from .append import _i32
from .mx import _call, _format_of
from .ops import _err_ptr

HEAD_DIMS = (64, 128, 256)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(*sizes: int) -> int:
    out = ctypes.c_int64()
    _native.check(_native.load().pace_kv_attention_workspace(*sizes, ctypes.byref(out)))
    return out.value


def _check(q: torch.Tensor, cache: torch.Tensor) -> int:
    """Validates queries and cache; returns the cache's format."""
    if cache.dim() != 5 or cache.shape[1] != 2 or not cache.is_contiguous() or not cache.is_cuda:
        raise ValueError("paged_kv_cache must be a contiguous device tensor [num_pages, 2, page_size, H, D] "
                         "(quantised: [..., row_width])")
    if q.dim() != 3 or q.dtype not in (torch.bfloat16, torch.float16) or q.device != cache.device:
        raise ValueError(f"q must be [nnz, num_qo_heads, head_dim] bfloat16 or float16 on {cache.device}")
    _, heads, D = q.shape
    if D not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {D}")
    if q.stride(2) != 1 or q.stride(1) != D:
        raise ValueError("q rows must be contiguous [num_qo_heads, head_dim] blocks")
    if cache.shape[3] == 0 or heads == 0 or heads % cache.shape[3]:
        raise ValueError(f"{heads} query heads do not divide over {cache.shape[3]} KV heads")
    if cache.dtype is torch.uint8:
        return _format_of(cache.shape[4], D)
    if cache.dtype != q.dtype or cache.shape[4] != D:
        raise ValueError(f"a cache of {cache.dtype} with head_dim {cache.shape[4]} for queries of {q.dtype} with {D}")
    return _native.PLAIN


def paged_attention(q: torch.Tensor, paged_kv_cache: torch.Tensor, kv_indices: torch.Tensor, kv_indptr: torch.Tensor,
                    kv_last_page_len: torch.Tensor, qo_indptr: Optional[torch.Tensor] = None, *,
                    max_q_len: Optional[int] = None, tree_mask: Optional[torch.Tensor] = None,
                    sm_scale: Optional[float] = None, logits_soft_cap: float = 0.0,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False,
                    err: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """softmax(scale * q k^T) v of each request's last tokens over its pages.

    q [nnz, num_qo_heads, head_dim] (bfloat16 or float16; head_dim 64, 128 or
    256; num_qo_heads a multiple of the cache's heads) holds the queries of
    request b in rows qo_indptr[b] .. qo_indptr[b + 1]; they are the request's
    last tokens, appended before the call.  Without qo_indptr each request has
    one.  max_q_len, needed with qo_indptr, bounds a request's queries; one with
    more is skipped and counted in `err`.

    A query sees every token before its request's queries, and of those: with
    tree_mask (int64 [nnz, words], bits) the j-th where bit j % 64 of word
    j // 64 of its row is set, else itself and those before it.  One that sees
    nothing gets zeros and a log-sum-exp of -inf.

    Scores and weighted sums are float32: a key whose products with a query
    pass its range upwards makes that query's row NaN, and values whose weighted
    sum passes it make the output infinite or NaN.  There is no backward pass:
    tensors that require gradients are refused while gradients are enabled.

    `err` goes up by one for each token on a page whose id is out of range (not
    read, not seen), each request whose offsets or last page's length are (cut),
    and each that is skipped, its rows not written.

    logits_soft_cap > 0 replaces scores s by cap * tanh(s / cap).  sm_scale is
    1 / sqrt(head_dim) by default.  Returns out ([nnz, num_qo_heads, head_dim],
    `out` if given; rows outside every request are not written), and with
    return_lse also the natural log-sum-exp [nnz, num_qo_heads] float32."""
    if torch.is_grad_enabled() and (q.requires_grad or paged_kv_cache.requires_grad):
        raise ValueError("paged_attention has no backward pass: call it under torch.no_grad() or with detached tensors")
    fmt = _check(q, paged_kv_cache)
    cache = paged_kv_cache
    dev, at = cache.device, cache.get_device()
    nnz, heads, D = q.shape
    num_pages, _, P, H, _ = cache.shape
    idx = _i32(kv_indices, "kv_indices", dev, at)
    ip = _i32(kv_indptr, "kv_indptr", dev, at)
    last = _i32(kv_last_page_len, "kv_last_page_len", dev, at)
    batch = last.numel()
    if ip.numel() != batch + 1:
        raise ValueError(f"kv_indptr needs {batch + 1} entries for {batch} requests")
    qo = None
    if qo_indptr is not None:
        qo = _i32(qo_indptr, "qo_indptr", dev, at)
        if qo.numel() != batch + 1:
            raise ValueError(f"qo_indptr needs {batch + 1} entries for {batch} requests")
        if max_q_len is None:
            raise ValueError("qo_indptr needs max_q_len, the most tokens that a request has")
        max_q_len = int(max_q_len)
        if max_q_len < 1:
            raise ValueError("max_q_len must be >= 1")
        max_q_len = min(max_q_len, max(nnz, 1))
    else:
        if nnz != batch:
            raise ValueError(f"without qo_indptr each request has one token: {nnz} for {batch} requests")
        if max_q_len not in (None, 1):
            raise ValueError("max_q_len needs qo_indptr")
        max_q_len = 1
    mask, words = None, 0
    if tree_mask is not None:
        if (tree_mask.dtype is not torch.int64 or tree_mask.dim() != 2 or tree_mask.shape[0] != nnz
                or tree_mask.device != dev or not tree_mask.is_contiguous()):
            raise ValueError(f"tree_mask must be a contiguous int64 tensor [{nnz}, words] on {dev}")
        words = tree_mask.shape[1]
        if 64 * words < max_q_len:
            raise ValueError(f"a tree_mask of {words} words holds {64 * words} tokens, max_q_len is {max_q_len}")
        mask = tree_mask.data_ptr()
    if sm_scale is None:
        sm_scale = 1 / math.sqrt(D)
    if not math.isfinite(sm_scale) or not math.isfinite(logits_soft_cap) or logits_soft_cap < 0:
        raise ValueError("sm_scale must be finite, logits_soft_cap finite and >= 0")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or out.stride(2) != 1 \
            or out.stride(1) != D:
        raise ValueError("out must be like q, its rows contiguous [num_qo_heads, head_dim] blocks")
    lse = torch.empty((nnz, heads), dtype=torch.float32, device=dev) if return_lse else None
    if nnz:
        sizes = (batch, H, heads // H, D, max_q_len, idx.numel(), P)
        need = _workspace_bytes(*sizes)
        # from torch's allocator on this stream: a captured graph gets its own
        space = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _call(dev, "pace_kv_attention", q.data_ptr(), q.stride(0) * 2 if nnz > 1 else heads * D * 2,
              _native.ELEM_TYPES[q.dtype], nnz, None if qo is None else qo.data_ptr(), batch, H, heads // H, D,
              cache.data_ptr(), fmt, num_pages, P, idx.data_ptr(), idx.numel(), ip.data_ptr(), last.data_ptr(),
              max_q_len, mask, words, sm_scale, logits_soft_cap, out.data_ptr(),
              out.stride(0) * 2 if nnz > 1 else heads * D * 2, None if lse is None else lse.data_ptr(),
              None if space is None else space.data_ptr(), need, _err_ptr(err))
    return (out, lse) if return_lse else out
