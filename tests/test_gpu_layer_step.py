"""The calls of a layer together, as a step makes them: tables, rows normalised,
rotated and written to the cache, attention over it.  Each result is checked
against the 64-bit oracles from what the call before it left in memory; pages
are found here by hand.  And latent pages moved like others."""
import math

import numpy as np
import pytest
import torch

from oracle import attention_oracle as ao
from oracle import rope_oracle as ro
from paceserve_amd.core.block_manager import NativeBlockAllocator
from paceserve_amd.kv_transfer import latent, migrate, mx, ops, rope
from paceserve_amd.kv_transfer.attention import paged_attention
from paceserve_amd.kv_transfer.swap import SwapSpace
from paceserve_amd.kv_transfer.tables import build_tables

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
EPS = 1e-6


def f64(x):
    return x.double().cpu().numpy()


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


def within(got, want, bound, what):
    got = f64(got)
    assert (np.abs(got - want) <= bound).all(), f"{what}: off by {np.max(np.abs(got - want) / bound):.3g} of its bound"


def check_rows(got, x, weight, positions, table, what):
    """Rows got [n, heads, D] of x at the positions."""
    x, t, eps = f64(x), f64(table), torch.finfo(got.dtype).eps
    for i, p in enumerate(positions):
        y, size = ro.turned(x[i], None if weight is None else f64(weight), EPS, t[p], False)
        within(got[i], y, ro.bound(y, size, x.shape[-1], eps, 2.0 ** -25 if got.dtype is FP16 else 0.0), f"{what} of token {i}")


def check_attention(out, lse, q, keys, values, scale, what):
    """One request's last tokens: out [T, Hq, Dv], values [n, H, Dv], Dv <= D."""
    D, Dv, eps = q.shape[2], out.shape[2], torch.finfo(out.dtype).eps
    n, sub = len(keys), 2.0 ** -25 if out.dtype is FP16 else 0.0
    wide = np.concatenate([values, np.zeros(values.shape[:2] + (D - Dv,))], 2)
    o, s, mean, dots, spread = ao.attend(f64(q), keys, wide, scale, 0.0, ao.visible(n, len(q), None))
    bo, bs = ao.bounds(D, eps, o, s, mean, dots, spread, 0.0, n, sub)
    within(out, o[..., :Dv], bo[..., :Dv], what)
    within(lse, s, bs, what + " (lse)")


class Pages:
    """A page table that a host fills: distinct pages in any order."""

    def __init__(self, rng, dev, batch, width, P, spare=5):
        self.num_pages, self.P, self.width = batch * width + spare, P, width
        self.ids = rng.permutation(self.num_pages)[:batch * width].reshape(batch, width).astype(np.int32)
        self.table = torch.from_numpy(self.ids).to(dev)

    def of(self, b, n):
        """(page, place) of request b's first n tokens."""
        at = np.arange(n)
        return self.ids[b, at // self.P].astype(np.int64), at % self.P


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("P,D,Hq,H,r", [(16, 128, 8, 2, 128), (24, 64, 3, 1, 32), (1, 128, 4, 4, 64)])
def test_prompts_then_single_tokens(gpu, P, D, Hq, H, r, dtype):
    rng = np.random.default_rng(P)
    new = [33, 1, 70, 16]
    batch, scale = len(new), 1 / math.sqrt(D)
    pages = Pages(rng, gpu, batch, -(-80 // P), P)
    cache = torch.zeros((pages.num_pages, 2, P, H, D), dtype=dtype, device=gpu)
    table = rope.rotary_table(100, r, device=gpu)
    w = torch.from_numpy(1 + 0.1 * rng.standard_normal(D)).to(dtype).to(gpu)
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    lens, held = np.zeros(batch, int), [np.zeros((0, H, D))] * batch     # the values that each request has
    for new in (new, [1, 1, 1, 1], [1, 1, 1, 1], [3, 0, 2, 1]):
        new = np.asarray(new)
        lens = lens + new
        qo, nnz = np.concatenate([[0], np.cumsum(new)]), int(new.sum())
        t = build_tables(pages.table, i32(lens, gpu), P, i32(qo, gpu), nnz + 2, err=err)
        qkv = torch.from_numpy(rng.standard_normal((nnz + 2, Hq + 2 * H, D))).to(dtype).to(gpu)
        q, k, v = qkv.split([Hq, H, H], 1)
        turned = rope.append_paged_kv_cache_rope(q, k, v, t.positions, t.slot_mapping, cache, table, w, w, eps=EPS, err=err)
        out, lse = paged_attention(turned, cache, t.kv_indices, t.kv_indptr, t.kv_last_page_len, i32(qo, gpu),
                                   max_q_len=int(new.max()), sm_scale=scale, return_lse=True, err=err)
        torch.cuda.synchronize()
        assert err.item() == 0
        for b in range(batch):
            at, n = slice(qo[b], qo[b + 1]), lens[b]
            positions = np.arange(n - new[b], n)
            page, place = pages.of(b, n)
            keys, values = cache[page, 0, place], f64(cache[page, 1, place])
            check_rows(turned[at], q[at], w, positions, table, f"queries of request {b}")
            check_rows(keys[n - new[b]:], k[at], w, positions, table, f"keys of request {b}")
            held[b] = np.concatenate([held[b], f64(v[at])])
            assert np.array_equal(values, held[b])
            if new[b]:
                check_attention(out[at], lse[at], turned[at], f64(keys), values, scale, f"request {b}")


@pytest.mark.parametrize("L,D,heads,P", [(256, 64, 4, 16), (512, 128, 3, 64), (256, 128, 2, 5)])
def test_latent_prompts_then_single_tokens(gpu, L, D, heads, P):
    """Head h's key and value are columns of the latent, so that expanding and
    absorbing round nothing: both forms answer the same question."""
    rng = np.random.default_rng(L + P)
    new = np.array([40, 1, 130])
    batch, scale = len(new), 1 / math.sqrt(D + 64)
    pages = Pages(rng, gpu, batch, -(-140 // P), P)
    cache = latent.empty_cache(pages.num_pages, P, L, device=gpu)
    table = rope.rotary_table(200, 64, device=gpu)
    w = torch.from_numpy(1 + 0.1 * rng.standard_normal(L)).to(BF16).to(gpu)
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    key_at = [(37 * h) % (L - D) for h in range(heads)]
    value_at = [(91 * h + 11) % (L - D) for h in range(heads)]
    lens = np.zeros(batch, int)
    for step, new in enumerate((new, np.ones(batch, int), np.array([2, 0, 3]))):
        lens = lens + new
        qo, nnz = np.concatenate([[0], np.cumsum(new)]), int(new.sum())
        t = build_tables(pages.table, i32(lens, gpu), P, i32(qo, gpu), nnz, err=err)
        down = torch.from_numpy(rng.standard_normal((nnz, L + 64))).to(BF16).to(gpu)
        latent.append_paged_latent_cache(down[:, :L], down[:, L:], t.positions, t.slot_mapping, cache, table, w, eps=EPS, err=err)
        q = torch.from_numpy(1.5 * rng.standard_normal((nnz, heads, D + 64))).to(BF16).to(gpu)
        given = q.clone()
        part = q[:, :, D:]                                # rotated in place, a slice of each head
        rope.norm_rotate(part, None, t.positions, table, out_q=part, err=err)
        absorbed = torch.zeros((nnz, heads, L + 64), dtype=BF16, device=gpu)
        absorbed[..., L:] = q[..., D:]
        for h in range(heads):
            absorbed[:, h, key_at[h]:key_at[h] + D] = q[:, h, :D]
        out, lse = latent.paged_latent_attention(absorbed, cache, t.kv_indices, t.kv_indptr, t.kv_last_page_len,
                                                 i32(qo, gpu), sm_scale=scale, max_q_len=int(new.max()), return_lse=True,
                                                 err=err)
        rows = [cache[torch.from_numpy(p).to(gpu), torch.from_numpy(s).to(gpu)] for p, s in
                (pages.of(b, lens[b]) for b in range(batch))]
        every = torch.cat(rows)
        ip = np.concatenate([[0], np.cumsum(lens)])
        key = torch.stack([every[:, a:a + D] for a in key_at], 1)
        value = torch.stack([every[:, a:a + D] for a in value_at], 1)
        expanded, lse2 = latent.latent_prompt_attention(q, key, every[:, L:], value, i32(qo, gpu), i32(ip, gpu),
                                                        return_lse=True, err=err)
        torch.cuda.synchronize()
        assert err.item() == 0 and torch.equal(q[..., :D], given[..., :D])
        for b in range(batch):
            at, n = slice(qo[b], qo[b + 1]), lens[b]
            positions = np.arange(n - new[b], n)
            x = rows[b][n - new[b]:]
            check_rows(x[:, None, L:], down[at, None, L:], None, positions, table, f"rotated part of request {b}")
            c = f64(down[at, :L])
            c = c / np.sqrt((c ** 2).mean(-1, keepdims=True) + EPS) * f64(w)
            within(x[:, :L], c, ro.bound(c, np.abs(c), L, 2.0 ** -7, 0.0), f"latents of request {b}")
            check_rows(part[at], given[at][..., D:], None, positions, table, f"queries of request {b}")
            if not new[b]:
                continue
            k = f64(rows[b])
            check_attention(out[at], lse[at], absorbed[at], k[:, None], k[:, None, :L], scale, f"absorbed, request {b}")
            for h in range(heads):
                keys = np.concatenate([k[:, key_at[h]:key_at[h] + D], k[:, L:]], 1)[:, None]
                check_attention(expanded[at, h:h + 1], lse2[at, h:h + 1], q[at, h:h + 1], keys,
                                k[:, None, value_at[h]:value_at[h] + D], scale, f"expanded, request {b} head {h}")


def test_a_captured_step_runs_on(gpu):
    """One graph of a decode step of both caches whose lengths advance on the GPU,
    replayed past pages' ends, with an unused place of the batch."""
    rng = np.random.default_rng(3)
    batch, P, D, Hq, H, L = 4, 4, 64, 4, 2, 256
    pages = Pages(rng, gpu, batch, 8, P)
    kv = torch.zeros((pages.num_pages, 2, P, H, mx.row_width(D, "mxfp8")), dtype=torch.uint8, device=gpu)
    rows = latent.empty_cache(pages.num_pages, P, L, device=gpu)
    twin_kv, twin_rows = kv.clone(), rows.clone()
    table = rope.rotary_table(64, 64, device=gpu)
    lens, grow = i32([3, 7, 0, 15], gpu), i32([1, 1, 0, 1], gpu)
    qkv = torch.zeros((batch, Hq + 2 * H, D), dtype=BF16, device=gpu)
    down = torch.zeros((batch, L + 64), dtype=BF16, device=gpu)
    q = torch.zeros((batch, Hq, L + 64), dtype=BF16, device=gpu)
    err = torch.zeros(1, dtype=torch.int32, device=gpu)

    def step(kv, rows, lens):
        t = build_tables(pages.table, lens, P, err=err)
        a, k, v = qkv.split([Hq, H, H], 1)
        turned = rope.append_paged_kv_cache_rope(a, k, v, t.positions, t.slot_mapping, kv, table, err=err)
        latent.append_paged_latent_cache(down[:, :L], down[:, L:], t.positions, t.slot_mapping, rows, table, err=err)
        return (paged_attention(turned, kv, t.kv_indices, t.kv_indptr, t.kv_last_page_len),
                latent.paged_latent_attention(q, rows, t.kv_indices, t.kv_indptr, t.kv_last_page_len, sm_scale=0.05))

    step(kv, rows, lens)                                  # warm
    kv.copy_(twin_kv)
    rows.copy_(twin_rows)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens.add_(grow)
        got = step(kv, rows, lens)
    now = np.array([3, 7, 0, 15])
    for _ in range(9):
        for x in (qkv, down, q):
            x.copy_(torch.from_numpy(rng.standard_normal(tuple(x.shape))).to(BF16))
        now = now + np.array([1, 1, 0, 1])
        graph.replay()
        torch.cuda.synchronize()
        want = step(twin_kv, twin_rows, i32(now, gpu))
        torch.cuda.synchronize()
        assert np.array_equal(lens.cpu().numpy(), now) and err.item() == 0
        assert torch.equal(kv, twin_kv) and torch.equal(rows.view(torch.int16), twin_rows.view(torch.int16))
        for a, b in zip(got, want):
            assert torch.equal(a, b) and (a[2] == 0).all()


@pytest.mark.parametrize("P,L,dtype", [(16, 512, BF16), (5, 256, FP16), (1, 512, BF16)])
def test_latent_pages_move_like_others(gpu, P, L, dtype):
    rng = np.random.default_rng(P)
    layers, num, lens = 3, 40, [5 * P, 3 * P - min(P - 1, 2), 1]
    src = [torch.from_numpy(rng.standard_normal((num, P, L + 64))).to(dtype).to(gpu) for _ in range(layers)]
    need = [-(-n // P) for n in lens]
    order, tables_, at = rng.permutation(num), [], 0
    for n in need:
        tables_.append(order[at:at + n].tolist())
        at += n
    q = torch.from_numpy(rng.standard_normal((3, 4, L + 64))).to(dtype).to(gpu)

    def answers(pool, tables):
        idx, ip = i32(np.concatenate(tables), gpu), i32(np.concatenate([[0], np.cumsum(need)]), gpu)
        last = i32([(n - 1) % P + 1 for n in lens], gpu)
        return [latent.paged_latent_attention(q, x, idx, ip, last, sm_scale=0.05) for x in pool]

    want = answers(src, tables_)
    pool = ops.PagedPool(src)
    assert pool.page_size == P and pool.page_shape == (P, L + 64) and pool.page_bytes == P * (L + 64) * 2
    for mode in ("fused", "buffer"):
        dst = [torch.zeros_like(x) for x in src]
        plan = migrate.KVMigrator(src, dst, NativeBlockAllocator(P, num, rng.permutation(num).tolist())).promote(tables_, mode=mode)
        for a, b in zip(answers(dst, plan.dst_tables), want):
            assert torch.equal(a, b)
        assert sum(int((x != 0).flatten(1).any(1).sum()) for x in dst) == layers * sum(need)
    # through a transfer buffer, and through host memory
    ids = sum(tables_, [])
    buf = ops.pack(src, ids)
    assert buf.shape == (layers, len(ids), P, L + 64)
    dst = [torch.zeros_like(x) for x in src]
    ops.unpack(buf, dst, list(range(len(ids))))
    near = [list(range(sum(need[:b]), sum(need[:b + 1]))) for b in range(3)]
    for a, b in zip(answers(dst, near), want):
        assert torch.equal(a, b)
    space = SwapSpace(dst, 16)
    for b, t in enumerate(near):
        space.swap_out(str(b), t)
    for x in dst:
        x.zero_()
    for b, t in enumerate(near):
        space.swap_in(str(b), [i + 20 for i in t])
    for a, b in zip(answers(dst, [[i + 20 for i in t] for t in near]), want):
        assert torch.equal(a, b)


def test_latent_pools_are_not_quantised_or_mixed(gpu):
    kept = latent.empty_cache(4, 16, 512, device=gpu)
    kv = torch.zeros((4, 2, 16, 2, 64), dtype=BF16, device=gpu)
    with pytest.raises(ValueError, match="latent"):
        mx.quantize_pages([kept], [0], [kept.view(torch.uint8)], [1])
    with pytest.raises(ValueError):
        ops.move([kept], [0], [kv], [0])
    with pytest.raises(ValueError):
        ops.PagedPool([kept, kv])
    with pytest.raises(ValueError):
        ops.PagedPool([torch.zeros((4, 1, 576), dtype=torch.uint8, device=gpu)[:, :, :568]])
