"""The tables of a batch built on the GPU (HIP): page lists end to end,
positions and cache slots, from the requests' lengths and a page table.

The host writes page ids into a request's row as it allocates them; what a step
needs follows from the lengths alone, so that a captured step can advance them
on the GPU.  The lists are the ones that the append and attention calls take
(paceserve/model_executor/attention/flashinfer_attention_wrapper.py:241-255).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .append import _i32
from .mx import _call
from .ops import _err_ptr


class BatchTables(NamedTuple):
    kv_indices: torch.Tensor        # int32 [num_indices], -1 behind the last request's pages
    kv_indptr: torch.Tensor         # int32 [batch + 1]
    kv_last_page_len: torch.Tensor  # int32 [batch]
    positions: torch.Tensor         # int32 [nnz], -1 for tokens of no request
    slot_mapping: torch.Tensor      # int64 [nnz], page * page_size + slot, or -1


def build_tables(page_table: torch.Tensor, seq_lens: torch.Tensor, page_size: int,
                 append_indptr: Optional[torch.Tensor] = None, nnz: Optional[int] = None, *,
                 num_indices: Optional[int] = None, out: Optional[BatchTables] = None,
                 err: Optional[torch.Tensor] = None) -> BatchTables:
    """Tables of requests whose first ceil(seq_lens[b] / page_size) pages are
    page_table[b] (int32 [batch, width], rows may be strided), and whose last
    append_indptr[b + 1] - append_indptr[b] tokens the step appends (without
    append_indptr: one each).

    nnz is the number of token rows (batch by default; needed with
    append_indptr): rows outside every request are padding, with position and
    slot -1.  num_indices is the length of kv_indices, width * batch by default;
    a captured step keeps it while the lengths change.  Attention divides its
    work, and sizes its workspace, by that length as if the requests filled it:
    give it what they may come to hold, not the table's room, where that is much
    more.  `out` takes the tables of an earlier call of the same sizes to write
    into.

    Sequence lengths are cut to [0, width * page_size], page lists to
    num_indices (kv_indptr runs on); a token before a request's first or past
    its pages gets slot -1.  A page id below 0 is a page that is not there yet:
    it is listed as it is, and its tokens get slot -1, which is padding to the
    appends; that is not counted here (attention counts the tokens on pages out
    of range that it should read).  `err` goes up by one for each request of which
    something is cut, whose offsets run backwards or leave [0, nnz], or that
    appends more tokens than it has (without append_indptr, one of length 0 is
    an unused place of the batch: no pages, position and slot -1)."""
    if page_table.dim() != 2 or page_table.dtype is not torch.int32 or not page_table.is_cuda \
            or (page_table.numel() > 0 and page_table.stride(1) != 1 and page_table.shape[1] > 1):
        raise ValueError("page_table must be an int32 device tensor [batch, width] with contiguous rows")
    dev, at = page_table.device, page_table.get_device()
    batch, width = page_table.shape
    if page_size < 1:
        raise ValueError("page_size must be >= 1")
    lens = _i32(seq_lens, "seq_lens", dev, at)
    if lens.numel() != batch:
        raise ValueError(f"{lens.numel()} sequence lengths for {batch} requests")
    ai = None
    if append_indptr is not None:
        ai = _i32(append_indptr, "append_indptr", dev, at)
        if ai.numel() != batch + 1:
            raise ValueError(f"append_indptr needs {batch + 1} entries for {batch} requests")
        if nnz is None:
            raise ValueError("append_indptr needs nnz, the number of token rows")
    elif nnz is None:
        nnz = batch
    nnz = int(nnz)
    if nnz < 0 or (ai is None and nnz < batch):
        raise ValueError(f"nnz must be at least the number of tokens, got {nnz}")
    if num_indices is None:
        num_indices = batch * width
    if num_indices < 0:
        raise ValueError("num_indices must be >= 0")
    sizes = ((num_indices, torch.int32), (batch + 1, torch.int32), (batch, torch.int32), (nnz, torch.int32),
             (nnz, torch.int64))
    if out is None:
        # two allocations instead of five: the call takes 9.8 us on the host, not 12.4
        ints = page_table.new_empty(num_indices + 2 * batch + 1 + nnz)
        out = BatchTables(*ints.split_with_sizes((num_indices, batch + 1, batch, nnz)),
                          page_table.new_empty(nnz, dtype=torch.int64))
    else:
        for name, t, (n, dtype) in zip(BatchTables._fields, out, sizes):
            if t.dtype is not dtype or t.dim() != 1 or t.numel() != n or t.device != dev or not t.is_contiguous():
                raise ValueError(f"out.{name} must be a contiguous {dtype} tensor of {n} entries on {dev}")
    _call(dev, "pace_kv_build_tables", page_table.data_ptr(), page_table.stride(0), width, lens.data_ptr(), batch,
          page_size, None if ai is None else ai.data_ptr(), nnz, out.kv_indices.data_ptr(), num_indices,
          out.kv_indptr.data_ptr(), out.kv_last_page_len.data_ptr(), out.positions.data_ptr(),
          out.slot_mapping.data_ptr(), _err_ptr(err))
    return out
