"""A quantised paged KV cache on the HIP path: appends that quantise the rows
they write, and conversion of whole pages between a 16- or 32-bit pool and a
quantised one.

Format.  Blocks of 32 elements along head_dim share one power-of-two scale, the
smallest 2^e that brings the block's largest magnitude within the element type:
e4m3 up to 448 ("mxfp8") or e2m1 up to 6 ("mxfp4").  An element is the value
times 2^-e, rounded to nearest even, and stands for its value whatever type it
is read as: float16 numbers from 57344 (mxfp4) or 63488 (mxfp8) on round to
65536, which float16 reads as infinity.  A block with an infinity or a NaN reads
as NaN.

A layer's cache is a contiguous uint8 tensor [num_pages, 2, page_size, H, R]
with R = row_width(D, format): D + D / 32 bytes for mxfp8, D / 2 + D / 32 for
mxfp4.  R and D together give the format, so no call takes it.  Within each
page half the elements [page_size, H, D] come first (4-bit ones two to a byte,
the even one low) and then the scale bytes [page_size, H, D / 32] (e + 127);
`elements_and_scales` gives both as views.  A page carries its scales: ops.pack,
move, swap, the channel and KVMigrator take such pools as they are, and move
half or a quarter of the bytes.

Pages of few tokens and heads can come to halves that are no multiple of 16
bytes (one token of one head of 128: 132 or 68).  rope.append_paged_kv_cache_rope
writes them; the appends and conversions here and attention.paged_attention
refuse them, and the calls that move pages those whose whole is none.

Like everything in this package the calls enqueue on the current stream and
return; tokens and pages with indices out of range are skipped and counted in
`err`.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _native
from .append import _i32
from .ops import IdsLike, PagedPool, _err_ptr, _stream_handle, as_pool, device_ids

BLOCK = 32
FORMATS = {"mxfp8": _native.MXFP8, "mxfp4": _native.MXFP4}


def row_width(head_dim: int, format: str) -> int:
    """Bytes per token and head, scales included."""
    if format not in FORMATS:
        raise ValueError(f"unknown format {format!r}: one of {', '.join(FORMATS)}")
    if head_dim <= 0 or head_dim % BLOCK:
        raise ValueError(f"head_dim ({head_dim}) must be a positive multiple of {BLOCK}")
    return (head_dim if format == "mxfp8" else head_dim // 2) + head_dim // BLOCK


def empty_cache(num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, format: str,
                device: Optional[torch.device] = None) -> torch.Tensor:
    """One layer's quantised cache, zeroed (zero bytes read as zeros)."""
    return torch.zeros((num_pages, 2, page_size, num_kv_heads, row_width(head_dim, format)), dtype=torch.uint8,
                       device="cuda" if device is None else device)


def _format_of(row: int, head_dim: int) -> int:
    """The format whose rows of head_dim elements take `row` bytes."""
    if head_dim > 0 and head_dim % BLOCK == 0:
        blocks = head_dim // BLOCK
        if row == 33 * blocks:
            return _native.MXFP8
        if row == 17 * blocks:
            return _native.MXFP4
    raise ValueError(f"rows of {row} bytes hold {head_dim} elements in no format: mxfp8 takes head_dim * 33 / 32 "
                     "bytes, mxfp4 head_dim * 17 / 32")


def elements_and_scales(cache: torch.Tensor, head_dim: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Views of a quantised cache [..., page_size, H, R]: element bytes [...,
    page_size, H, D or D / 2] and scale bytes [..., page_size, H, D / 32]."""
    _format_of(cache.shape[-1], head_dim)
    P, H, R = cache.shape[-3:]
    width = R - head_dim // BLOCK
    flat = cache.flatten(-3)
    return (flat[..., :P * H * width].unflatten(-1, (P, H, width)),
            flat[..., P * H * width:].unflatten(-1, (P, H, head_dim // BLOCK)))


def _call(device: torch.device, name: str, *args) -> None:
    """A library call on the device that its tensors are on."""
    fn = getattr(_native.load(), name)
    if device.index == torch.cuda.current_device():
        _native.check(fn(*args, _stream_handle(device)))
    else:
        with torch.cuda.device(device):
            _native.check(fn(*args, _stream_handle(device)))


def _append_format(key: torch.Tensor, value: torch.Tensor, cache: torch.Tensor) -> int:
    """The format of an append's cache.  One look at each property settles an
    append that is in order; any other gets _check_append's checks and message."""
    if type(cache) is type(key) is type(value) is torch.Tensor and cache.dtype is torch.uint8:
        index, shape, rows, stride, dtype = cache.get_device(), cache.shape, key.shape, key.stride(), key.dtype
        if (index >= 0 and len(shape) == 5 and len(rows) == 3 and shape[1] == 2 and rows[1] == shape[3]
                and stride[2] == 1 and stride[1] == rows[2] and value.shape == rows and value.stride() == stride
                and value.dtype is dtype and dtype in _native.ELEM_TYPES and cache.is_cuda
                and key.get_device() == value.get_device() == index and cache.is_contiguous()):
            return _format_of(shape[4], rows[2])
    _check_append(key, value, cache)
    return _format_of(cache.shape[4], key.shape[2])


def _check_append(key: torch.Tensor, value: torch.Tensor, cache: torch.Tensor) -> None:
    """Validates the rows and the quantised cache."""
    if cache.dtype is not torch.uint8 or cache.dim() != 5 or cache.shape[1] != 2 or not cache.is_contiguous() \
            or not cache.is_cuda:
        raise ValueError("mx_cache must be a contiguous uint8 device tensor [num_pages, 2, page_size, H, row_width]")
    H, dev = cache.shape[3], cache.device
    for name, t in (("append_key", key), ("append_value", value)):
        if t.dim() != 3 or t.shape[1] != H or t.device != dev or t.dtype not in _native.ELEM_TYPES:
            raise ValueError(f"{name} must be [nnz, {H}, head_dim] bfloat16, float16 or float32 on {dev}")
        if t.stride(2) != 1 or t.stride(1) != t.shape[2]:
            raise ValueError(f"{name} rows must be contiguous [H, D] blocks")
    if key.shape != value.shape or key.dtype != value.dtype or key.stride(0) != value.stride(0):
        raise ValueError("append_key and append_value differ in shape, dtype or token stride")


def append_paged_kv_cache_mx(append_key: torch.Tensor, append_value: torch.Tensor, batch_indices: torch.Tensor,
                             positions: torch.Tensor, mx_cache: torch.Tensor, kv_indices: torch.Tensor,
                             kv_indptr: torch.Tensor, kv_last_page_len: torch.Tensor,
                             err: Optional[torch.Tensor] = None) -> None:
    """append.append_paged_kv_cache into a quantised cache: the rows
    ([nnz, H, D] bfloat16, float16 or float32) are quantised as they are
    written.  Tokens of one call take distinct slots."""
    fmt = _append_format(append_key, append_value, mx_cache)
    dev, at, nnz = mx_cache.device, mx_cache.get_device(), append_key.shape[0]
    bi = _i32(batch_indices, "batch_indices", dev, at)
    pos = _i32(positions, "positions", dev, at)
    idx = _i32(kv_indices, "kv_indices", dev, at)
    ip = _i32(kv_indptr, "kv_indptr", dev, at)
    _i32(kv_last_page_len, "kv_last_page_len", dev, at)
    if bi.numel() < nnz or pos.numel() < nnz:
        raise ValueError("batch_indices and positions need one entry per appended token")
    if nnz == 0:
        return
    _, H, D = append_key.shape
    _call(dev, "pace_kv_append_mx", append_key.data_ptr(), append_value.data_ptr(),
          _native.ELEM_TYPES[append_key.dtype], append_key.stride(0) * append_key.element_size(), nnz, bi.data_ptr(),
          pos.data_ptr(), ip.numel() - 1, mx_cache.data_ptr(), fmt, mx_cache.shape[0], idx.data_ptr(), idx.numel(),
          ip.data_ptr(), mx_cache.shape[2], H * D, _err_ptr(err))


def append_paged_kv_cache_mx_indptr(append_key: torch.Tensor, append_value: torch.Tensor,
                                    append_indptr: torch.Tensor, mx_cache: torch.Tensor, kv_indices: torch.Tensor,
                                    kv_indptr: torch.Tensor, kv_last_page_len: torch.Tensor,
                                    err: Optional[torch.Tensor] = None) -> None:
    """append.append_paged_kv_cache_indptr into a quantised cache: one launch
    that also derives each token's request and position."""
    fmt = _append_format(append_key, append_value, mx_cache)
    dev, at, nnz = mx_cache.device, mx_cache.get_device(), append_key.shape[0]
    ai = _i32(append_indptr, "append_indptr", dev, at)
    idx = _i32(kv_indices, "kv_indices", dev, at)
    ip = _i32(kv_indptr, "kv_indptr", dev, at)
    last = _i32(kv_last_page_len, "kv_last_page_len", dev, at)
    batch = ai.numel() - 1
    if ip.numel() != batch + 1 or last.numel() != batch:
        raise ValueError(f"kv_indptr needs {batch + 1} entries and kv_last_page_len {batch} for {batch} requests")
    if nnz == 0:
        return
    _, H, D = append_key.shape
    _call(dev, "pace_kv_append_mx_indptr", append_key.data_ptr(), append_value.data_ptr(),
          _native.ELEM_TYPES[append_key.dtype], append_key.stride(0) * append_key.element_size(), nnz, ai.data_ptr(),
          batch, mx_cache.data_ptr(), fmt, mx_cache.shape[0], idx.data_ptr(), idx.numel(), ip.data_ptr(),
          last.data_ptr(), mx_cache.shape[2], H * D, _err_ptr(err))


def _pools(plain, small) -> Tuple[PagedPool, PagedPool, int]:
    pp, sp = as_pool(plain), as_pool(small)
    if pp.host or sp.host:
        raise ValueError("quantised pages convert between device pools")
    if len(pp.page_shape) != 4 or len(sp.page_shape) != 4:
        raise ValueError("quantised pages are those of keys and values: a latent cache has none")
    if pp.dtype not in _native.ELEM_TYPES:
        raise ValueError(f"pool of {pp.dtype}: bfloat16, float16 or float32 is converted")
    if sp.dtype is not torch.uint8:
        raise ValueError(f"a quantised pool is uint8, got {sp.dtype}")
    if pp.page_shape[:3] != sp.page_shape[:3] or pp.num_layers != sp.num_layers or pp.device != sp.device:
        raise ValueError("source and destination pools differ in page size, heads, layers or device")
    return pp, sp, _format_of(sp.page_shape[3], pp.page_shape[3])


def _convert(name: str, src: PagedPool, src_ids: IdsLike, src_kind: int, dst: PagedPool, dst_ids: IdsLike,
             dst_kind: int, half: int, layer_begin: int, layer_end: Optional[int], err) -> None:
    lb, le = src.layer_range(layer_begin, layer_end)
    s_ids = device_ids(src_ids, src.device)
    d_ids = device_ids(dst_ids, dst.device, distinct=True)
    n = s_ids.numel()
    if n != d_ids.numel():
        raise ValueError(f"{n} source ids but {d_ids.numel()} destination ids")
    if n == 0 or le == lb:
        return
    _call(src.device, name, src.table(lb), src.num_pages, s_ids.data_ptr(), src_kind, dst.table(lb), dst.num_pages,
          d_ids.data_ptr(), dst_kind, le - lb, n, half, _err_ptr(err))


def quantize_pages(src, src_ids: IdsLike, dst, dst_ids: IdsLike, *, layer_begin: int = 0,
                   layer_end: Optional[int] = None, err: Optional[torch.Tensor] = None) -> None:
    """dst.layers[l][dst_ids[j]] = src.layers[l][src_ids[j]] quantised: whole
    pages of a bfloat16, float16 or float32 pool into a quantised one, as
    ops.move moves them between like pools.  dst_ids must be distinct."""
    pp, sp, fmt = _pools(src, dst)
    P, H, D = pp.page_shape[1:]
    _convert("pace_kv_quantize_pages", pp, src_ids, _native.ELEM_TYPES[pp.dtype], sp, dst_ids, fmt, P * H * D,
             layer_begin, layer_end, err)


def dequantize_pages(src, src_ids: IdsLike, dst, dst_ids: IdsLike, *, layer_begin: int = 0,
                     layer_end: Optional[int] = None, err: Optional[torch.Tensor] = None) -> None:
    """dst.layers[l][dst_ids[j]] = the values of the quantised page
    src.layers[l][src_ids[j]], rounded to dst's type (past its range:
    infinity).  dst_ids must be distinct."""
    pp, sp, fmt = _pools(dst, src)
    P, H, D = pp.page_shape[1:]
    _convert("pace_kv_dequantize_pages", sp, src_ids, fmt, pp, dst_ids, _native.ELEM_TYPES[pp.dtype], P * H * D,
             layer_begin, layer_end, err)
