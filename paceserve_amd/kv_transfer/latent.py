"""A paged cache of latent vectors on the HIP path, its writer, and attention
over it: absorbed (every head reads the cached row itself) for single and
drafted tokens, expanded (each head has keys and values of its own) for prompts.

A model with latent attention keeps one row a token and layer, [latent, key
part]: latent_dim numbers that stand for all heads' keys and values, and 64 that
are the rotated part of every head's key.  A layer's cache is
[num_pages, page_size, latent_dim + 64] in bfloat16 or float16, with the page
ids and tables of the other caches; ops, swap, the channel and KVMigrator move
such pages as they move others.

With W_k and W_v the matrices that expand a latent c to a head's key and value:
q . (W_k c) = (W_k^T q) . c, so a query multiplied by W_k^T once attends to the
rows as they are, and the weighted sum of latents, multiplied by W_v, is the
head's output.  That reads the least per token, which is what a decode step
pays for; a prompt has enough queries for its keys and values to be expanded
first, which is a third of the products.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Tuple, Union

import torch

from .. import _native
from .append import _i32
from .mx import _call
from .ops import _err_ptr
from .rope import ROW_TYPES, _check_table, _check_weight, _i64, _refuse_gradients

ROPE_DIM = 64
LATENT_DIMS = (256, 512)
PROMPT_HEAD_DIMS = (64, 128)


def empty_cache(num_pages: int, page_size: int, latent_dim: int, dtype: torch.dtype = torch.bfloat16,
                device: Optional[torch.device] = None) -> torch.Tensor:
    """One layer's latent cache, zeroed."""
    if latent_dim not in LATENT_DIMS:
        raise ValueError(f"latent_dim must be one of {LATENT_DIMS}, got {latent_dim}")
    if dtype not in ROW_TYPES:
        raise ValueError(f"a latent cache is bfloat16 or float16, got {dtype}")
    return torch.zeros((num_pages, page_size, latent_dim + ROPE_DIM), dtype=dtype,
                       device="cuda" if device is None else device)


def _check_cache(cache: torch.Tensor) -> int:
    """Validates a latent cache; returns latent_dim."""
    if cache.dim() != 3 or not cache.is_contiguous() or not cache.is_cuda or cache.dtype not in ROW_TYPES \
            or cache.shape[2] - ROPE_DIM not in LATENT_DIMS:
        raise ValueError("latent_cache must be a contiguous bfloat16 or float16 device tensor [num_pages, page_size, "
                         f"latent_dim + {ROPE_DIM}] with latent_dim one of {LATENT_DIMS}")
    return cache.shape[2] - ROPE_DIM


def append_paged_latent_cache(latent: torch.Tensor, rope_key: torch.Tensor, positions: torch.Tensor,
                              slot_mapping: torch.Tensor, latent_cache: torch.Tensor, table: torch.Tensor,
                              weight: Optional[torch.Tensor] = None, *, eps: float = 1e-6, interleaved: bool = False,
                              err: Optional[torch.Tensor] = None) -> None:
    """Writes each token's row [latent', rope_key'] to its slot: latent'
    [nnz, latent_dim] normalised as in rope.norm_rotate where there is a weight
    [latent_dim], rope_key' [nnz, 64] rotated by the table's (rotary_dim 64) row
    of the token's position.

    The rows may be slices of one projection (token strides of a multiple of 16
    bytes).  slot_mapping[i] = page * page_size + slot (int64, as
    tables.build_tables gives it); tokens of one call take distinct slots.  A
    token with slot -1 is padding; one with another slot outside the cache, or a
    position outside the table, is counted in `err` and not written.  There is
    no backward pass."""
    _refuse_gradients("append_paged_latent_cache", latent, rope_key, weight, latent_cache)
    L = _check_cache(latent_cache)
    dev, nnz = latent_cache.device, latent.shape[0] if latent.dim() else -1
    for name, x, dim in (("latent", latent, L), ("rope_key", rope_key, ROPE_DIM)):
        if x.shape != (nnz, dim) or x.dtype is not latent_cache.dtype or x.device != dev \
                or (nnz > 0 and x.stride(1) != 1):
            raise ValueError(f"{name} must be [nnz, {dim}] {latent_cache.dtype} rows on {dev}")
    pos, slots = _i32(positions, "positions", dev, latent_cache.get_device()), _i64(slot_mapping, "slot_mapping", dev)
    if pos.numel() != nnz or slots.numel() != nnz:
        raise ValueError(f"{pos.numel()} positions and {slots.numel()} slots for {nnz} tokens")
    rows, rotary = _check_table(table, dev)
    if rotary != ROPE_DIM:
        raise ValueError(f"the table must rotate {ROPE_DIM} columns, not {rotary}")
    w = _check_weight("weight", weight, latent_cache, L)
    _call(dev, "pace_kv_append_latent", latent.data_ptr(), latent.stride(0) * 2 if nnz > 1 else 0, rope_key.data_ptr(),
          rope_key.stride(0) * 2 if nnz > 1 else 0, w, _native.ELEM_TYPES[latent_cache.dtype], L, nnz, pos.data_ptr(),
          slots.data_ptr(), table.data_ptr(), rows, interleaved, eps, latent_cache.data_ptr(), latent_cache.shape[0],
          latent_cache.shape[1], _err_ptr(err))


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(*sizes: int) -> int:
    out = ctypes.c_int64()
    _native.check(_native.load().pace_kv_latent_attention_workspace(*sizes, ctypes.byref(out)))
    return out.value


def paged_latent_attention(q: torch.Tensor, latent_cache: torch.Tensor, kv_indices: torch.Tensor,
                           kv_indptr: torch.Tensor, kv_last_page_len: torch.Tensor,
                           qo_indptr: Optional[torch.Tensor] = None, *, sm_scale: float,
                           max_q_len: Optional[int] = None, tree_mask: Optional[torch.Tensor] = None,
                           out: Optional[torch.Tensor] = None, return_lse: bool = False,
                           err: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """The absorbed form: softmax(sm_scale * q . row) latent of each request's
    last tokens over its pages.

    q [nnz, num_heads, latent_dim + 64] holds each head's query multiplied by
    W_k^T, then its rotated part.  sm_scale is the model's, 1 / sqrt of a head's
    expanded key.  Returns out [nnz, num_heads, latent_dim] (`out` if given), the
    weighted sums of latents, for W_v; with return_lse also the natural
    log-sum-exp [nnz, num_heads] float32.

    Tables, qo_indptr, max_q_len, tree_mask, rows that see nothing, rows outside
    every request, `err` and captured calls are as in attention.paged_attention.
    There is no backward pass."""
    _refuse_gradients("paged_latent_attention", q, latent_cache)
    cache = latent_cache
    L = _check_cache(cache)
    dev, at = cache.device, cache.get_device()
    if q.dim() != 3 or q.dtype is not cache.dtype or q.device != dev or q.shape[2] != L + ROPE_DIM or q.shape[1] == 0:
        raise ValueError(f"q must be [nnz, num_heads, {L + ROPE_DIM}] {cache.dtype} on {dev}")
    nnz, heads, W = q.shape
    if nnz > 0 and (q.stride(2) != 1 or (heads > 1 and q.stride(1) != W)):
        raise ValueError("q rows must be contiguous [num_heads, latent_dim + 64] blocks")
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
    if not math.isfinite(sm_scale):
        raise ValueError("sm_scale must be finite")
    if out is None:
        out = torch.empty((nnz, heads, L), dtype=q.dtype, device=dev)
    elif out.shape != (nnz, heads, L) or out.dtype is not q.dtype or out.device != dev \
            or (nnz > 0 and (out.stride(2) != 1 or (heads > 1 and out.stride(1) != L))):
        raise ValueError(f"out must be [{nnz}, {heads}, {L}] {q.dtype} on {dev}, its rows contiguous "
                         "[num_heads, latent_dim] blocks")
    lse = torch.empty((nnz, heads), dtype=torch.float32, device=dev) if return_lse else None
    if nnz:
        need = _workspace_bytes(batch, heads, L, max_q_len, idx.numel(), cache.shape[1])
        # from torch's allocator on this stream: a captured graph gets its own
        space = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _call(dev, "pace_kv_latent_attention", q.data_ptr(), q.stride(0) * 2 if nnz > 1 else heads * W * 2,
              _native.ELEM_TYPES[q.dtype], nnz, None if qo is None else qo.data_ptr(), batch, heads, L, cache.data_ptr(),
              cache.shape[0], cache.shape[1], idx.data_ptr(), idx.numel(), ip.data_ptr(), last.data_ptr(), max_q_len,
              mask, words, sm_scale, out.data_ptr(), out.stride(0) * 2 if nnz > 1 else heads * L * 2,
              None if lse is None else lse.data_ptr(), None if space is None else space.data_ptr(), need, _err_ptr(err))
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=4096)
def _prompt_workspace_bytes(*sizes: int) -> int:
    out = ctypes.c_int64()
    _native.check(_native.load().pace_kv_prompt_attention_workspace(*sizes, ctypes.byref(out)))
    return out.value


def latent_prompt_attention(q: torch.Tensor, key: torch.Tensor, rope_key: torch.Tensor, value: torch.Tensor,
                            qo_indptr: torch.Tensor, kv_indptr: torch.Tensor, *, sm_scale: Optional[float] = None,
                            max_q_len: Optional[int] = None, causal: bool = True, out: Optional[torch.Tensor] = None,
                            return_lse: bool = False,
                            err: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """The expanded form: softmax(sm_scale * q . [key, rope_key]) value of ragged
    prompts, over keys and values that the caller expanded from the latents.

    q [nnz, num_heads, D + 64] (D 64 or 128; the last 64 columns rotated), key
    and value [num_keys, num_heads, D], rope_key [num_keys, 64], which all heads
    share.  Request b has queries qo_indptr[b] .. qo_indptr[b + 1] and keys
    kv_indptr[b] .. kv_indptr[b + 1]; its queries are its last tokens.  causal:
    query i of q_len sees the keys up to kv_len - q_len + i; otherwise all of its
    request's.  Tensors may be slices of wider ones (token and head strides of a
    multiple of 16 bytes, keys' and values' tokens less than 64 MiB apart): key
    and value of one projection.

    sm_scale is 1 / sqrt(D + 64) by default.  Returns out [nnz, num_heads, D]
    (`out` if given; rows outside every request are not written), and with
    return_lse also the natural log-sum-exp [nnz, num_heads] float32.  A query
    that sees nothing gets zeros and -inf.  `err` goes up by one for each request
    that is skipped (queries outside the rows or more than max_q_len, nnz by
    default) or whose key offsets run backwards or leave the keys (cut to them).
    There is no backward pass."""
    _refuse_gradients("latent_prompt_attention", q, key, rope_key, value)
    if q.dim() != 3 or q.dtype not in ROW_TYPES or not q.is_cuda or q.shape[2] - ROPE_DIM not in PROMPT_HEAD_DIMS \
            or q.shape[1] == 0:
        raise ValueError("q must be a bfloat16 or float16 device tensor [nnz, num_heads, D + 64] with D one of "
                         f"{PROMPT_HEAD_DIMS}")
    dev, at = q.device, q.get_device()
    nnz, heads, width = q.shape
    D = width - ROPE_DIM
    n = key.shape[0] if key.dim() else -1
    for name, x, shape in (("key", key, (n, heads, D)), ("value", value, (n, heads, D)), ("rope_key", rope_key, (n, ROPE_DIM))):
        if x.shape != shape or x.dtype is not q.dtype or x.device != dev:
            raise ValueError(f"{name} must be {list(shape)} {q.dtype} on {dev}")
    for name, x in (("q", q), ("key", key), ("value", value), ("rope_key", rope_key)):
        if x.numel() > 0 and x.stride(-1) != 1:
            raise ValueError(f"{name} must have contiguous columns")
    qo = _i32(qo_indptr, "qo_indptr", dev, at)
    ip = _i32(kv_indptr, "kv_indptr", dev, at)
    batch = qo.numel() - 1
    if batch < 0 or ip.numel() != batch + 1:
        raise ValueError("qo_indptr and kv_indptr need one entry more than there are requests")
    if max_q_len is None:
        max_q_len = max(nnz, 1)
    if max_q_len < 1:
        raise ValueError("max_q_len must be >= 1")
    if sm_scale is None:
        sm_scale = 1 / math.sqrt(width)
    if not math.isfinite(sm_scale):
        raise ValueError("sm_scale must be finite")
    if out is None:
        out = torch.empty((nnz, heads, D), dtype=q.dtype, device=dev)
    elif out.shape != (nnz, heads, D) or out.dtype is not q.dtype or out.device != dev \
            or (nnz > 0 and out.stride(2) != 1):
        raise ValueError(f"out must be [{nnz}, {heads}, {D}] {q.dtype} on {dev} with contiguous columns")
    lse = torch.empty((nnz, heads), dtype=torch.float32, device=dev) if return_lse else None

    def strides(x):
        return x.stride(0) * 2 if x.shape[0] > 1 else 0, x.stride(1) * 2 if heads > 1 else 0

    if nnz:
        need = _prompt_workspace_bytes(nnz, n, batch, heads, D, int(causal))
        space = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _call(dev, "pace_kv_prompt_attention", q.data_ptr(), *strides(q), key.data_ptr(), *strides(key),
              rope_key.data_ptr(), rope_key.stride(0) * 2 if n > 1 else 0, value.data_ptr(), *strides(value),
              _native.ELEM_TYPES[q.dtype], heads, D, nnz, n, qo.data_ptr(), ip.data_ptr(), batch,
              min(int(max_q_len), max(nnz, 1)), sm_scale, causal, out.data_ptr(), *strides(out),
              None if lse is None else lse.data_ptr(), None if space is None else space.data_ptr(), need, _err_ptr(err))
    return (out, lse) if return_lse else out
