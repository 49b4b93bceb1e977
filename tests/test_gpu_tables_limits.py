"""build_tables (HIP) over page tables with holes, and the calls that take its tables."""
import numpy as np
import pytest
import torch

from paceserve_amd.kv_transfer import latent, rope
from paceserve_amd.kv_transfer.attention import paged_attention
from paceserve_amd.kv_transfer.tables import build_tables

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


def test_pages_that_are_not_there_yet(gpu):
    """Their tokens are padding to the appends, which nobody counts; attention counts what it
    should read of them."""
    P, table = 4, np.array([[3, 5, -1], [0, -7, 2], [1, 4, 6]])
    lens, qo = [9, 10, 7], [0, 3, 9, 10]
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    t = build_tables(i32(table, gpu), i32(lens, gpu), P, i32(qo, gpu), 12, err=err)
    assert err.item() == 0
    assert t.kv_indices.tolist() == [3, 5, -1, 0, -7, 2, 1, 4, -1] and t.kv_indptr.tolist() == [0, 3, 6, 8]
    assert t.kv_last_page_len.tolist() == [1, 2, 3]
    assert t.positions.tolist() == [6, 7, 8, 4, 5, 6, 7, 8, 9, 6, -1, -1]
    # request 0: 6, 7 on page 5, 8 on none; 1: 4 to 7 on none, 8, 9 on page 2; 2: 6 on page 4
    assert t.slot_mapping.tolist() == [22, 23, -1, -1, -1, -1, -1, 8, 9, 18, -1, -1]
    there = np.array(t.slot_mapping.tolist()) >= 0
    x = torch.randn((12, 4, 64), generator=torch.Generator().manual_seed(0)).to(BF16).to(gpu)
    angles = rope.rotary_table(16, 64, device=gpu)
    cache = torch.zeros((7, 2, P, 1, 64), dtype=BF16, device=gpu)
    out = torch.full((12, 2, 64), 7.0, dtype=BF16, device=gpu)
    rope.append_paged_kv_cache_rope(x[:, :2], x[:, 2:3], x[:, 3:], t.positions, t.slot_mapping, cache, angles, out=out, err=err)
    rows = latent.empty_cache(7, P, 256, device=gpu)
    latent.append_paged_latent_cache(x.view(12, 256), x[:, 0], t.positions, t.slot_mapping, rows, angles, err=err)
    assert err.item() == 0
    assert ((out == 7).flatten(1).all(1).cpu().numpy() == ~there).all()
    assert (cache[:, 1] != 0).flatten(2).any(2).sum() == there.sum() == (rows != 0).any(2).sum()
    q = torch.randn((10, 2, 64), generator=torch.Generator().manual_seed(1)).to(BF16).to(gpu)
    args = (t.kv_indices, t.kv_indptr, t.kv_last_page_len, i32(qo, gpu))
    paged_attention(q, cache, *args, max_q_len=6, err=err)
    assert err.item() == 1 + 4
    wide = torch.zeros((10, 2, 320), dtype=BF16, device=gpu)
    latent.paged_latent_attention(wide, rows, *args, sm_scale=0.1, max_q_len=6, err=err)
    assert err.item() == 10
