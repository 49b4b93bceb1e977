"""Queries and keys normalised per head and rotated by position on the HIP
path, into tensors or, with the values, straight into a paged cache.

The step between a layer's projection and its attention: what
append.append_paged_kv_cache (and mx's) take already normalised and rotated,
these take as projected
(paceserve/model_executor/attention/flashinfer_attention_wrapper.py:241-255).
Rows are bfloat16 or float16, the arithmetic is float32, rounded once.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _native
from .append import _i32
from .mx import _call, _format_of
from .ops import _err_ptr

ROW_TYPES = (torch.bfloat16, torch.float16)


def rotary_table(num_positions: int, rotary_dim: int, base: float = 10000.0,
                 device: Optional[torch.device] = None) -> torch.Tensor:
    """float32 [num_positions, rotary_dim]: of each position t the cosines of
    t * base^(-2 i / rotary_dim), i < rotary_dim / 2, then the sines.  Angles
    are float64, so far positions keep theirs.  A model with scaled frequencies
    brings a table of its own in the same layout."""
    if num_positions < 0 or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("num_positions must be >= 0, rotary_dim positive and even")
    dev = torch.device("cuda" if device is None else device)
    i = torch.arange(0, rotary_dim, 2, device=dev, dtype=torch.float64)
    angle = torch.arange(num_positions, device=dev, dtype=torch.float64)[:, None] * base ** (-i / rotary_dim)
    return torch.cat([torch.cos(angle), torch.sin(angle)], 1).float()


def _refuse_gradients(name: str, *tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} has no backward pass: call it under torch.no_grad() or with detached tensors")


def _i64(t: torch.Tensor, name: str, dev: torch.device) -> torch.Tensor:
    if t.dtype is torch.int64 and t.dim() == 1 and t.get_device() == dev.index and t.is_contiguous():
        return t
    if t.dim() != 1 or t.device != dev:
        raise ValueError(f"{name} must be a 1-D tensor on {dev}")
    if t.dtype is torch.int64 and t.is_contiguous():
        return t
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be int64 or int32, got {t.dtype}")
    return t.to(torch.int64).contiguous()


def _check_table(table: torch.Tensor, dev: torch.device) -> Tuple[int, int]:
    if table.dim() != 2 or table.dtype is not torch.float32 or table.device != dev or not table.is_contiguous():
        raise ValueError(f"table must be a contiguous float32 tensor [num_positions, rotary_dim] on {dev}")
    return table.shape[0], table.shape[1]


def _check_rows(name: str, x: torch.Tensor, like: torch.Tensor, heads: Optional[int] = None) -> None:
    """Rows [nnz, heads, D] of like's length, head size and type, each head's columns contiguous."""
    # One look at each property settles a good tensor (a decode step's append 14.1 to 12.5 us
    # on the host, with the others like this).
    if heads is not None or x is like:
        want = like.shape if heads is None else (like.shape[0], heads, like.shape[2])
        if x.shape == want and x.dtype is like.dtype and x.get_device() == like.get_device() and x.stride(2) == 1:
            return
    if x.dim() != 3 or x.shape[0] != like.shape[0] or x.shape[2] != like.shape[2] or x.dtype is not like.dtype \
            or x.device != like.device or (heads is not None and x.shape[1] != heads):
        raise ValueError(f"{name} must be [{like.shape[0]}, {'heads' if heads is None else heads}, {like.shape[2]}] "
                         f"{like.dtype} on {like.device}")
    if x.numel() > 0 and x.stride(2) != 1:
        raise ValueError(f"{name} must have contiguous columns")


def _check_weight(name: str, w: Optional[torch.Tensor], x: torch.Tensor, dim: int) -> Optional[int]:
    if w is None:
        return None
    if w.shape != (dim,) or w.dtype is not x.dtype or w.device != x.device or not w.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {x.dtype} tensor of {dim} entries on {x.device}")
    return w.data_ptr()


def _strides(x: torch.Tensor) -> Tuple[int, int]:
    """Bytes between tokens and between heads; where there is one of them, its stride says nothing."""
    nnz, heads, dim = x.shape
    token, head, _ = x.stride()
    return token * 2 if nnz > 1 else 0, head * 2 if heads > 1 else dim * 2


def _turn_args(name: str, q: torch.Tensor, positions: torch.Tensor, table: torch.Tensor):
    """(positions, table's rows, rotary_dim), checked."""
    if q.dtype not in ROW_TYPES or not q.is_cuda:
        raise ValueError(f"{name} takes bfloat16 or float16 device rows")
    dev = q.device
    pos = _i32(positions, "positions", dev, dev.index)
    if pos.numel() != q.shape[0]:
        raise ValueError(f"{pos.numel()} positions for {q.shape[0]} tokens")
    rows, rotary = _check_table(table, dev)
    return pos, rows, rotary


def norm_rotate(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, table: torch.Tensor,
                q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, *,
                eps: float = 1e-6, interleaved: bool = False, out_q: Optional[torch.Tensor] = None,
                out_k: Optional[torch.Tensor] = None,
                err: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(q', k'): each head of q [nnz, num_qo_heads, D] and k [nnz, num_kv_heads, D]
    (or None) as x / sqrt(mean(x^2) + eps) * weight where there is a weight [D],
    then its first rotary_dim columns rotated by the table's row of the token's
    position (rotary_table): columns (i, i + rotary_dim / 2), or (2 i, 2 i + 1)
    if interleaved, take the angle of position and i.

    D and rotary_dim are multiples of 16; rows may be strided slices of a
    projection, each head 16-byte aligned.  out_q and out_k may be q and k
    themselves; otherwise they share no memory with them.  A token whose position is outside the table is counted in `err`
    and its rows are not written.  Squares are float32 sums: rows past 2^64
    normalise to zeros.  There is no backward pass."""
    _refuse_gradients("norm_rotate", q, k, q_weight, k_weight)
    if q.dim() != 3:
        raise ValueError("q must be [nnz, num_qo_heads, head_dim]")
    _check_rows("q", q, q)
    pos, rows, rotary = _turn_args("norm_rotate", q, positions, table)
    if k is not None:
        _check_rows("k", k, q)
    elif k_weight is not None or out_k is not None:
        raise ValueError("k_weight and out_k need k")
    D = q.shape[2]
    qw, kw = _check_weight("q_weight", q_weight, q, D), _check_weight("k_weight", k_weight, q, D)
    if out_q is None:
        out_q = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _check_rows("out_q", out_q, q, q.shape[1])
    if k is not None:
        if out_k is None:
            out_k = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        else:
            _check_rows("out_k", out_k, k, k.shape[1])
        k_args = (k.data_ptr(), *_strides(k), k.shape[1], out_k.data_ptr(), *_strides(out_k), kw)
    else:
        k_args = (None, 0, 0, 0, None, 0, 0, None)
    _call(q.device, "pace_kv_norm_rotate", q.data_ptr(), *_strides(q), q.shape[1], out_q.data_ptr(), *_strides(out_q),
          qw, *k_args, _native.ELEM_TYPES[q.dtype], D, q.shape[0], pos.data_ptr(), table.data_ptr(), rows, rotary,
          interleaved, eps, _err_ptr(err))
    return out_q, out_k


def append_paged_kv_cache_rope(query: torch.Tensor, append_key: torch.Tensor, append_value: torch.Tensor,
                               positions: torch.Tensor, slot_mapping: torch.Tensor, paged_kv_cache: torch.Tensor,
                               table: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                               k_weight: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                               interleaved: bool = False, out: Optional[torch.Tensor] = None,
                               err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """norm_rotate of query and append_key, with the keys and append_value
    ([nnz, num_kv_heads, D]) written to their slots of a layer's cache in the
    same pass; returns the queries (`out` if given, which may be `query`).

    slot_mapping[i] = page * page_size + slot (int64, as tables.build_tables
    gives it); tokens of one call take distinct slots.  The cache is of the
    rows' type, [num_pages, 2, page_size, num_kv_heads, D], or quantised (mx;
    D and rotary_dim then in multiples of 64, pages of any size): its elements
    are rounded once, from the float32 results.

    A token with slot -1 is padding: nothing of it is written.  One with another
    slot outside the cache, or a position outside the table, is counted in `err`
    and not written."""
    cache = paged_kv_cache
    _refuse_gradients("append_paged_kv_cache_rope", query, append_key, append_value, q_weight, k_weight, cache)
    if query.dim() != 3:
        raise ValueError("query must be [nnz, num_qo_heads, head_dim]")
    _check_rows("query", query, query)
    pos, rows, rotary = _turn_args("append_paged_kv_cache_rope", query, positions, table)
    if cache.dim() != 5 or cache.shape[1] != 2 or not cache.is_contiguous() or cache.device != query.device:
        raise ValueError("paged_kv_cache must be a contiguous device tensor [num_pages, 2, page_size, H, D] "
                         "(quantised: [..., row_width])")
    num_pages, _, P, H, width = cache.shape
    D = query.shape[2]
    _check_rows("append_key", append_key, query, H)
    _check_rows("append_value", append_value, query, H)
    if cache.dtype is torch.uint8:
        fmt = _format_of(width, D)
    elif cache.dtype is query.dtype and width == D:
        fmt = _native.PLAIN
    else:
        raise ValueError(f"a cache of {cache.dtype} with head_dim {width} for rows of {query.dtype} with {D}")
    slots = _i64(slot_mapping, "slot_mapping", query.device)
    if slots.numel() != query.shape[0]:
        raise ValueError(f"{slots.numel()} slots for {query.shape[0]} tokens")
    qw, kw = _check_weight("q_weight", q_weight, query, D), _check_weight("k_weight", k_weight, query, D)
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    else:
        _check_rows("out", out, query, query.shape[1])
    # Few tokens of few heads: half a quantised page is no multiple of 16 bytes.
    name = "pace_kv_append_rope" if fmt == _native.PLAIN or P * H * width % 16 == 0 else "pace_kv_append_rope_packed"
    _call(query.device, name, query.data_ptr(), *_strides(query), query.shape[1], out.data_ptr(),
          *_strides(out), qw, append_key.data_ptr(), *_strides(append_key), kw, append_value.data_ptr(),
          *_strides(append_value), H, _native.ELEM_TYPES[query.dtype], D, query.shape[0], pos.data_ptr(),
          slots.data_ptr(), table.data_ptr(), rows, rotary, interleaved, eps, cache.data_ptr(), fmt, num_pages, P,
          _err_ptr(err))
    return out
