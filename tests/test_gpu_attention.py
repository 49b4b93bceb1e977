"""paged_attention (HIP) against the 64-bit oracle.

Every result is held to a bound made from the numbers themselves (oracle.
attention_oracle.bounds): the roundings that the kernel's arithmetic makes, none
of them measured."""
import math

import numpy as np
import pytest
import torch

from oracle import attention_oracle as ao
from oracle import mx_oracle as mo
from paceserve_amd.kv_transfer import append as ap
from paceserve_amd.kv_transfer import mx, ops
from paceserve_amd.kv_transfer.attention import paged_attention
from paceserve_amd.kv_transfer.migrate import KVMigrator
from paceserve_amd.core.block_manager import BlockAllocator

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


class Batch:
    """Requests of `kv` tokens whose last `new` are queries, on permuted pages;
    every byte that no request's token owns is a NaN's (or 0xFF)."""

    def __init__(self, dev, kv, new, *, H=2, G=4, D=128, P=16, dtype=BF16, fmt=None, tree=False, seed=0, q_gain=1.5,
                 spare=3):
        rng = self.rng = np.random.default_rng(seed)
        kv, new = np.asarray(kv), np.asarray(new)
        self.dev, self.kv, self.new, self.H, self.G, self.D, self.P = dev, kv, new, H, G, D, P
        self.dtype, self.fmt = dtype, fmt
        pages = -(-kv // P)
        self.num_pages = int(pages.sum()) + spare
        self.indptr = np.concatenate([[0], np.cumsum(pages)])
        self.indices = rng.permutation(self.num_pages)[:self.indptr[-1]]
        self.last = np.where(kv == 0, 0, (kv - 1) % P + 1)
        self.qo = np.concatenate([[0], np.cumsum(new)])
        self.nnz = int(self.qo[-1])
        self.rows = [torch.from_numpy(rng.standard_normal((n, 2, H, D)) * np.exp(0.5 * rng.standard_normal((2, H, D))))
                     for n in kv]
        self.q = torch.from_numpy(q_gain * rng.standard_normal((self.nnz, H * G, D))).to(dtype).to(dev)
        words = max(1, -(-int(max(new, default=1)) // 64))
        self.mask = None
        if tree:
            m = np.zeros((self.nnz, words), np.uint64)
            for b, t in enumerate(new):
                for i in range(t):
                    row = self.qo[b] + i
                    if i:
                        m[row] = m[self.qo[b] + i - 1 - rng.integers(0, min(i, 8))]
                    m[row, i // 64] |= np.uint64(1 << (i % 64))
            self.mask = m
        self.fill()

    def fill(self):
        """Writes self.rows into a fresh cache."""
        P, H, D = self.P, self.H, self.D
        if self.fmt is None:
            cache = torch.full((self.num_pages, 2, P, H, D), math.nan, dtype=self.dtype)
        else:
            cache = torch.full((self.num_pages, 2, P, H, mx.row_width(D, self.fmt)), 255, dtype=torch.uint8)
            data, byte = mx.elements_and_scales(cache, D)
        self.seen_rows = []
        for b, x in enumerate(self.rows):
            pos = np.arange(len(x))
            page = torch.from_numpy(self.indices[self.indptr[b] + pos // P].astype(np.int64))
            slot = torch.from_numpy(pos % P)
            if self.fmt is None:
                cache[page, :, slot] = x.to(self.dtype)
                self.seen_rows.append(x.to(self.dtype).double().numpy())
            else:
                codes, c = mo.quantize(x.float().double().numpy(), self.fmt)
                packed = mo.pack(codes, self.fmt)
                data[page, :, slot], byte[page, :, slot] = torch.from_numpy(packed), torch.from_numpy(c)
                with np.errstate(over="ignore"):
                    self.seen_rows.append(torch.from_numpy(mo.values(packed, c, self.fmt)).to(self.dtype).double()
                                          .numpy())
        self.cache = cache.to(self.dev)

    def tables(self):
        return i32(self.indices, self.dev), i32(self.indptr, self.dev), i32(self.last, self.dev)

    def device_mask(self):
        return None if self.mask is None else torch.from_numpy(self.mask.view(np.int64)).to(self.dev)

    def run(self, cap=0.0, **more):
        qo = i32(self.qo, self.dev)
        return paged_attention(self.q, self.cache, *self.tables(), qo, max_q_len=max(1, int(self.new.max())),
                               tree_mask=self.device_mask(), logits_soft_cap=cap, return_lse=True, **more)

    def check(self, out, lse, cap=0.0, hidden=None, scale=None):
        scale = 1 / math.sqrt(self.D) if scale is None else scale
        got_o, got_l = out.double().cpu().numpy(), lse.double().cpu().numpy()
        eps = torch.finfo(self.dtype).eps
        sub = 2.0 ** -25 if self.dtype is FP16 else 0.0
        for b, x in enumerate(self.seen_rows):
            n, t, r = len(x), int(self.new[b]), slice(self.qo[b], self.qo[b + 1])
            if t == 0:
                continue
            sees = ao.visible(n, t, None if self.mask is None else self.mask[r])
            if hidden is not None:
                sees &= ~hidden(b, np.arange(n))[None, :]
            o, s, mean, dots, spread = ao.attend(self.q[r].double().cpu().numpy(), x[:, 0], x[:, 1], scale, cap, sees)
            bo, bs = ao.bounds(self.D, eps, o, s, mean, dots, spread, cap, n, sub)
            # Scores are float32 sums: a row whose sum of |q k| passes 2^128 (a key of
            # bfloat16's lowest value, -1.99 * 2^127, does with any sum of |q| over 1)
            # has no score there, and nothing is said about it.
            within = np.isnan(dots) | (np.abs(dots) < 2.0 ** 128 * abs(scale))
            for x64 in (o, s, bo, bs, got_o[r], got_l[r]):
                x64[~within] = 0
            assert np.array_equal(np.isnan(o), np.isnan(got_o[r])), f"request {b}: NaN in other places"
            fine = np.isfinite(o)
            assert (np.abs(got_o[r] - o)[fine] <= bo[fine]).all(), \
                f"request {b}: out off by {np.max((np.abs(got_o[r] - o) / bo)[fine]):.3g} of its bound"
            dead = np.isneginf(s)
            assert np.array_equal(dead, np.isneginf(got_l[r])) and (got_o[r][dead] == 0).all()
            ok = np.isfinite(s)
            assert (np.abs(got_l[r] - s)[ok] <= bs[ok]).all(), f"request {b}: lse off"


CASES = [
    # kv lengths, queries, H, G, D, P
    ([1], [1], 1, 1, 128, 16),
    ([16, 17, 31, 1, 300], [1] * 5, 2, 4, 128, 16),
    ([700, 33, 5], [1, 1, 1], 8, 8, 64, 16),
    ([513, 64], [1, 1], 2, 16, 256, 16),
    ([40, 9, 130], [5, 9, 2], 2, 4, 128, 16),
    ([100, 64, 63], [33, 64, 1], 1, 1, 64, 24),
    ([300, 70], [12, 70], 2, 3, 128, 7 * 16),
    ([5000, 260], [3, 3], 2, 4, 128, 16),
    ([4097], [21], 1, 7, 256, 32),
    ([0, 20, 0, 7], [0, 4, 0, 0], 2, 2, 64, 16),
    ([257, 400], [129, 200], 1, 2, 128, 1 * 64),
    ([90] * 70, [1] * 70, 1, 4, 128, 16),
]


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dtype,fmt", [(BF16, None), (FP16, None), (BF16, "mxfp8"), (FP16, "mxfp8"), (BF16, "mxfp4"),
                                       (FP16, "mxfp4")])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_matches_the_oracle(gpu, case, dtype, fmt, tree):
    kv, new, H, G, D, P = CASES[case]
    print(f"attention case {case} {dtype} {fmt} tree={tree}", flush=True)
    b = Batch(gpu, kv, new, H=H, G=G, D=D, P=P, dtype=dtype, fmt=fmt, tree=tree, seed=case)
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    cap = 20.0 if case % 3 == 2 else 0.0
    out, lse = b.run(cap, err=err)
    torch.cuda.synchronize()
    b.check(out, lse, cap)
    assert err.item() == 0


def test_one_token_form_is_the_same(gpu):
    b = Batch(gpu, [300, 1, 17], [1, 1, 1])
    out, lse = b.run()
    o2, l2 = paged_attention(b.q, b.cache, *b.tables(), return_lse=True)
    assert torch.equal(out, o2) and torch.equal(lse, l2)
    b.check(o2, l2)


@pytest.mark.parametrize("dtype,fmt", [(BF16, None), (FP16, None), (BF16, "mxfp8")])
@pytest.mark.parametrize("T,G", [(6, 2), (20, 8)])
def test_what_is_not_seen_cannot_matter(gpu, dtype, fmt, T, G):
    """Drafted tokens with infinities, NaN and the type's lowest values: rows
    that see them get what the definition gives, the others are untouched."""
    b = Batch(gpu, [50, 200], [T, T], dtype=dtype, fmt=fmt, tree=True, G=G, seed=3)
    low = float(torch.finfo(dtype).min)
    for x, n in zip(b.rows, b.kv):
        first = n - T
        x[first + 2, 1, 0, 5] = math.inf
        x[first + 3, 0, 1, 7] = math.nan
        x[first + 4, 1] = math.nan
        x[first + 5, 0] = low
        x[first + 5, 1, :, 3] = low
    # token 1 sees none of them, token 2 sees only itself beside the context
    for r in range(2):
        for i in range(T):
            own = 1 << i
            b.mask[b.qo[r] + i, 0] = np.uint64(own | (1 if i % 2 else 0) | (4 if i == 5 else 0))
    b.fill()
    out, lse = b.run()
    torch.cuda.synchronize()
    b.check(out, lse)
    assert torch.isfinite(out[b.qo[0] + 1]).all() and torch.isfinite(out[b.qo[1] + 6 - 6]).all()


def test_rows_that_see_nothing(gpu):
    b = Batch(gpu, [4, 30], [4, 4], tree=True, seed=1)
    b.mask[1] = 0                                       # no context and no bit: nothing
    b.mask[5] = 0                                       # a context of 26 tokens
    out, lse = b.run()
    b.check(out, lse)
    assert (out[1] == 0).all() and torch.isneginf(lse[1]).all() and torch.isfinite(lse[5]).all()


def test_scores_of_the_lowest_value_and_wide_scores(gpu):
    """Scores thousands apart, and a scale of zero and a negative one."""
    b = Batch(gpu, [200, 40], [2, 3], seed=2, q_gain=300.0)
    out, lse = b.run()
    b.check(out, lse)
    for scale in (0.0, -0.1):
        out, lse = b.run(sm_scale=scale)
        torch.cuda.synchronize()
        got = out.double().cpu().numpy()
        for r, x in enumerate(b.seen_rows):
            s = slice(b.qo[r], b.qo[r + 1])
            o, _, mean, dots, spread = ao.attend(b.q[s].double().cpu().numpy(), x[:, 0], x[:, 1], scale, 0.0,
                                                 ao.visible(len(x), int(b.new[r]), None))
            bo, _ = ao.bounds(b.D, torch.finfo(BF16).eps, o, o[..., 0], mean, np.abs(dots), spread, 0.0, len(x), 0.0)
            assert (np.abs(got[s] - o) <= bo).all()


@pytest.mark.parametrize("fmt", [None, "mxfp8"])
def test_bad_pages_and_requests_are_skipped(gpu, fmt):
    b = Batch(gpu, [100, 90, 64], [3, 5, 2], fmt=fmt, seed=4)
    b.indices = b.indices.copy()
    b.indices[2], b.indices[b.indptr[1]] = b.num_pages, -5        # tokens 32..47 of request 0, 0..15 of request 1
    out, lse = b.run()
    torch.cuda.synchronize()
    b.check(out, lse, hidden=lambda r, p: (p // 16 == 2) if r == 0 else (p // 16 == 0) if r == 1 else p < 0)
    # a request with more queries than max_q_len is left alone and counted
    b = Batch(gpu, [100, 90, 64], [3, 5, 2], fmt=fmt, seed=4)
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    out = torch.full_like(b.q, 7.0)
    paged_attention(b.q, b.cache, *b.tables(), i32(b.qo, gpu), max_q_len=4, out=out, err=err)
    assert err.item() == 1 and (out[3:8] == 7).all()
    full, _ = b.run()
    assert torch.equal(out[:3], full[:3]) and torch.equal(out[8:], full[8:])


def test_rows_behind_the_last_request_are_left(gpu):
    b = Batch(gpu, [100, 90], [3, 5], seed=5)
    want, _ = b.run()
    q = torch.cat([b.q, torch.full_like(b.q[:4], math.nan)])
    out = torch.full_like(q, 5.0)
    paged_attention(q, b.cache, *b.tables(), i32(b.qo, gpu), max_q_len=5, out=out)
    assert torch.equal(out[:8], want) and (out[8:] == 5).all()


def test_strided_queries_and_output(gpu):
    b = Batch(gpu, [100, 290], [3, 5], seed=6)
    want, _ = b.run()
    wide = torch.full((8, 14, 128), math.nan, dtype=BF16, device=gpu)
    wide[:, 2:10] = b.q
    room = torch.full((8, 9, 128), 3.0, dtype=BF16, device=gpu)
    out = paged_attention(wide[:, 2:10], b.cache, *b.tables(), i32(b.qo, gpu), max_q_len=8, out=room[:, 1:])
    # max_q_len only bounds the requests' queries: rows are the same rows
    assert out.data_ptr() == room[:, 1:].data_ptr() and (room[:, 0] == 3).all()
    np.testing.assert_allclose(room[:, 1:].float().cpu().numpy(), want.float().cpu().numpy(), rtol=2 ** -7, atol=2e-2)


def test_results_repeat_bit_for_bit(gpu):
    b = Batch(gpu, [6000, 3000], [4, 2], seed=7, H=1)
    first, l1 = b.run()
    for _ in range(3):
        again, l2 = b.run()
        assert torch.equal(first, again) and torch.equal(l1, l2)


def test_graph_replays_follow_the_tables(gpu):
    """Captured once, replayed over changed lengths, pages and queries, two
    graphs and eager calls in turn."""
    b = Batch(gpu, [5000, 700], [4, 4], seed=8, tree=True)
    idx, ip, last = b.tables()
    qo, mask = i32(b.qo, gpu), b.device_mask()

    def call():
        return paged_attention(b.q, b.cache, idx, ip, last, qo, max_q_len=4, tree_mask=mask, return_lse=True)

    call()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = call()
        graphs.append((graph, res))
    for step in range(4):
        b.q.copy_(torch.randn_like(b.q))
        if step:
            ip.copy_(i32([0, 300 - 90 * step, b.indptr[-1]], gpu))      # fewer pages, more to the second request
            last.copy_(i32([5, 3 + step], gpu))
        # slots past the old lengths hold NaN, so only pages filled to their end are given out
        with torch.no_grad():
            b.cache.copy_(torch.nan_to_num(b.cache, nan=0.25))
        want = call()
        torch.cuda.synchronize()
        for graph, res in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, res in graphs:
            assert torch.equal(res[0], want[0]) and torch.equal(res[1], want[1])


def test_calls_on_two_streams(gpu):
    b, c = Batch(gpu, [5000], [3], seed=9), Batch(gpu, [4000], [2], seed=10, fmt="mxfp4")
    want, other = b.run()[0], c.run()[0]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(5):
        for s, x in zip(streams, (b, c)):
            with torch.cuda.stream(s):
                got.append(x.run()[0])
    torch.cuda.synchronize()
    for k, g in enumerate(got):
        assert torch.equal(g, want if k % 2 == 0 else other)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_a_request_lives_through_all_of_them(gpu, fmt):
    """A prompt prefilled in bf16 is handed over quantised, drafted tokens are
    appended quantised, the tree is attended to, the request moves to another
    pool and is read back: each step against the oracle on the bytes before it."""
    H, G, D, P, L, n, T = 2, 4, 128, 16, 2, 75, 5
    rng = np.random.default_rng(11)
    plain = [torch.from_numpy(rng.standard_normal((9, 2, P, H, D))).to(BF16).to(gpu) for _ in range(L)]
    small = [mx.empty_cache(9, P, H, D, fmt, gpu) for _ in range(L)]
    table = [4, 0, 7, 2, 5]
    mx.quantize_pages(plain, [8, 1, 3, 6, 0], small, table)
    new = torch.from_numpy(rng.standard_normal((T, 2 * H, D))).to(BF16).to(gpu)
    q = torch.from_numpy(rng.standard_normal((T, H * G, D))).to(BF16).to(gpu)
    mask = torch.tensor([[1], [3], [5], [11], [21]], dtype=torch.int64, device=gpu)
    tables = i32(table, gpu), i32([0, 5], gpu), i32([(n - 1) % P + 1], gpu)
    for c in small:
        mx.append_paged_kv_cache_mx_indptr(new[:, :H], new[:, H:], i32([0, T], gpu), c, *tables)
    there = [torch.zeros_like(c) for c in small]
    mig = KVMigrator(ops.PagedPool(small), ops.PagedPool(there), BlockAllocator(P, 9))
    plan = mig.promote([table], mode="fused")
    moved = i32(plan.dst_tables[0][:5], gpu), tables[1], tables[2]
    back = [torch.zeros_like(p) for p in plain]
    mx.dequantize_pages(there, moved[0], back, i32([0, 1, 2, 3, 4], gpu))
    for l in range(L):
        out, lse = paged_attention(q, there[l], *moved, i32([0, T], gpu), max_q_len=T, tree_mask=mask,
                                   return_lse=True)
        same = paged_attention(q, small[l], *tables, i32([0, T], gpu), max_q_len=T, tree_mask=mask)
        assert torch.equal(out, same)
        # rows from their definition: quantised prompt, quantised drafts
        rows = plain[l][[8, 1, 3, 6, 0]].double().cpu().numpy().transpose(0, 2, 1, 3, 4).reshape(-1, 2, H, D)[:n]
        rows[n - T:] = new.double().cpu().numpy().reshape(T, 2, H, D)
        codes, byte = mo.quantize(rows, fmt)
        rows = mo.values(mo.pack(codes, fmt), byte, fmt)
        read = back[l][:5].double().cpu().numpy().transpose(0, 2, 1, 3, 4).reshape(-1, 2, H, D)[:n]
        assert np.array_equal(read, rows)
        o, s, mean, dots, spread = ao.attend(q.double().cpu().numpy(), rows[:, 0], rows[:, 1], 1 / math.sqrt(D), 0.0,
                                             ao.visible(n, T, mask.cpu().numpy().view(np.uint64)))
        bo, bs = ao.bounds(D, torch.finfo(BF16).eps, o, s, mean, dots, spread, 0.0, n, 0.0)
        assert (np.abs(out.double().cpu().numpy() - o) <= bo).all()
        assert (np.abs(lse.double().cpu().numpy() - s) <= bs).all()


def test_python_refusals(gpu):
    b = Batch(gpu, [40, 20], [3, 2])
    t, qo = b.tables(), i32(b.qo, gpu)
    mask = torch.zeros((5, 1), dtype=torch.int64, device=gpu)

    def bad(msg, q=b.q, cache=b.cache, tables=t, qo_indptr=qo, **kw):
        kw.setdefault("max_q_len", 3)
        with pytest.raises(ValueError, match=msg):
            paged_attention(q, cache, *tables, qo_indptr, **kw)

    bad("contiguous device", cache=b.cache.cpu())
    bad("contiguous device", cache=b.cache[:, :, ::2])
    bad("q must be", q=b.q.float())
    bad("q must be", q=b.q.cpu())
    bad("head_dim must", q=torch.zeros(5, 8, 96, dtype=BF16, device=gpu))
    bad("contiguous \\[num", q=b.q.transpose(0, 1))
    bad("do not divide", q=b.q[:, :7].contiguous())
    bad("a cache of", cache=b.cache.half())
    bad("no format", cache=b.cache.view(torch.uint8))
    bad("kv_indptr needs", tables=(t[0], t[1][:2], t[2]))
    bad("qo_indptr needs", qo_indptr=qo[:2])
    bad("needs max_q_len", max_q_len=None)
    bad(">= 1", max_q_len=0)
    bad("one token", qo_indptr=None, max_q_len=None)
    bad("tree_mask must", tree_mask=mask.int())
    bad("tree_mask must", tree_mask=mask[:4])
    bad("words holds", tree_mask=mask[:, :0])
    bad("finite", sm_scale=math.inf)
    bad("finite", logits_soft_cap=-1.0)
    bad("out must", out=b.q.float())
    bad("is on cpu", tables=(t[0].cpu(), t[1], t[2]))
    empty = paged_attention(b.q[:0], b.cache, t[0][:0], i32([0], gpu), t[2][:0], i32([0], gpu), max_q_len=1)
    assert empty.shape == (0, 8, 128)


def test_pages_of_one_and_three_tokens(gpu):
    for P, D, fmt in ((1, 128, None), (3, 64, None), (1, 256, "mxfp8"), (16, 64, "mxfp4")):
        b = Batch(gpu, [70, 1, 131], [3, 1, 2], H=2, G=2, D=D, P=P, fmt=fmt, seed=12)
        out, lse = b.run()
        torch.cuda.synchronize()
        b.check(out, lse)


@pytest.mark.parametrize("R", [256, 257, 700])
def test_many_requests(gpu, R):
    """More requests than one round of the search takes, some without tokens."""
    rng = np.random.default_rng(R)
    kv, new = rng.integers(1, 40, R), rng.integers(0, 3, R)
    new = np.minimum(new, kv)
    b = Batch(gpu, kv, new, H=1, G=2, D=64, seed=R)
    out, lse = b.run()
    torch.cuda.synchronize()
    b.check(out, lse)


@pytest.mark.parametrize("G,T,n", [(1, 1, 40000), (2, 2, 36000), (12, 40, 3000)])
def test_many_chunks(gpu, G, T, n):
    """More chunks of a request than a wave weighs at once, and more rows than the
    joining workgroups take one by one (12 * 40 * 8 heads)."""
    b = Batch(gpu, [n, 100], [T, 1], H=8 if n == 3000 else 1, G=G, D=64, seed=n, tree=n == 3000)
    out, lse = b.run()
    torch.cuda.synchronize()
    b.check(out, lse)


def test_fewer_tokens_than_queries(gpu):
    """Queries whose own place lies before the first token see nothing."""
    b = Batch(gpu, [2, 0, 30, 0], [5, 3, 2, 1], seed=13)
    out, lse = b.run()
    torch.cuda.synchronize()
    b.check(out, lse)
    assert (out[:3] == 0).all() and (out[5:8] == 0).all() and torch.isneginf(lse[5:8]).all()
    none = Batch(gpu, [0, 0], [1, 1], seed=13)             # no pages at all
    out, lse = none.run()
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_requests_share_pages(gpu):
    """Two requests whose tables name the same pages (a shared prefix), and a mask
    with more words than the tokens need."""
    b = Batch(gpu, [100, 90], [3, 4], seed=14, tree=True)
    b.indices = b.indices.copy()
    b.indices[b.indptr[1]:b.indptr[1] + 5] = b.indices[:5]
    b.seen_rows[1] = np.concatenate([b.seen_rows[0][:80], b.seen_rows[1][80:]])
    b.mask = np.concatenate([b.mask, np.full((7, 2), 2 ** 64 - 1, np.uint64)], 1)
    out, lse = b.run()
    torch.cuda.synchronize()
    b.check(out, lse)


@pytest.mark.parametrize("fmt", [None, "mxfp8"])
def test_offsets_past_32_bits(gpu, fmt):
    """A layer's cache of more than 4 GiB, its last pages in use: appended to,
    converted, attended to."""
    H, D, P = 8, 128, 64
    width = D if fmt is None else mx.row_width(D, fmt)
    pages = (9 << 29) // (2 * P * H * width * (2 if fmt is None else 1)) + 8
    b = Batch(gpu, [150, 70], [4, 2], H=H, G=2, D=D, P=P, fmt=fmt, seed=15)
    cache = torch.zeros((pages, 2, P, H, width), dtype=b.cache.dtype, device=gpu)
    assert cache.numel() * cache.element_size() > 1 << 32
    move = pages - b.num_pages
    cache[move:] = b.cache
    small, b.cache = b.cache, cache
    b.indices = b.indices + move
    out, lse = b.run()
    torch.cuda.synchronize()
    b.check(out, lse)
    if fmt is not None:
        plain = [torch.zeros((b.num_pages, 2, P, H, D), dtype=BF16, device=gpu) for _ in range(2)]
        every = list(range(b.num_pages))
        mx.dequantize_pages([cache], [move + i for i in every], plain[:1], every)
        mx.dequantize_pages([small], every, plain[1:], every)
        assert torch.equal(plain[0].view(torch.int16), plain[1].view(torch.int16))
        mx.quantize_pages(plain[:1], [2], [cache], [pages - 1])
        mx.quantize_pages(plain[:1], [2], [small], [b.num_pages - 1])
        rows = torch.randn(3, H, D, device=gpu, dtype=BF16)
        for c, at in ((cache, pages - 2), (small, b.num_pages - 2)):
            mx.append_paged_kv_cache_mx_indptr(rows, rows, i32([0, 3], gpu), c, i32([at], gpu), i32([0, 1], gpu),
                                               i32([7], gpu))
        assert torch.equal(cache[move:], small) and not cache[:move].any()


@pytest.mark.parametrize("seed", range(24))
def test_random_batches(gpu, seed):
    rng = np.random.default_rng(1000 + seed)
    R = int(rng.integers(1, 9))
    D = int(rng.choice([64, 128, 256]))
    fmt = [None, "mxfp8", "mxfp4"][int(rng.integers(3))]
    kv = rng.integers(0, int(rng.choice([20, 200, 2500])) + 1, R)
    new = np.minimum(rng.integers(0, int(rng.choice([1, 6, 80])) + 1, R), np.maximum(kv, 0))
    new[0] = max(new[0], 1)
    kv[0] = max(kv[0], 1)
    case = dict(H=int(rng.integers(1, 4)), G=int(rng.choice([1, 2, 3, 5, 8])), D=D, P=int(rng.choice([16, 16, 32, 48])),
                dtype=[BF16, FP16][int(rng.integers(2))], fmt=fmt, tree=bool(rng.integers(2)), seed=seed)
    print(f"random batch {kv.tolist()} {new.tolist()} {case}", flush=True)
    b = Batch(gpu, kv, new, **case)
    cap = float(rng.choice([0.0, 15.0]))
    out, lse = b.run(cap)
    torch.cuda.synchronize()
    b.check(out, lse, cap)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("chunks", [2, 3, 5, 17, 18, 63, 64, 65, 66, 67, 69, 71, 127, 130])
def test_every_count_of_chunks(gpu, D, chunks):
    """A long context over few pages, named again and again: as many chunks of 512
    tokens, the last one short, as the joining waves may get, alone and split."""
    b = Batch(gpu, [8 * 16], [1], H=1, G=1, D=D, seed=chunks)
    n = 512 * (chunks - 1) + 17
    table = np.arange(-(-n // 16)) % 8
    rows = b.seen_rows[0].reshape(8, 16, 2, 1, D)
    b.seen_rows[0] = np.ascontiguousarray(rows[table].reshape(-1, 2, 1, D)[:n])
    b.indices, b.indptr, b.last = b.indices[table], np.array([0, len(table)]), np.array([(n - 1) % 16 + 1])
    out, lse = b.run()
    torch.cuda.synchronize()
    b.check(out, lse)


def test_offsets_that_run_backwards(gpu):
    """kv_indptr [0, 200, 0, 200] counts every page twice: more work items than the call has room for.  The
    first request is whole, the second has no pages, the third is refused."""
    b = Batch(gpu, [3200, 0, 0], [1, 0, 0], H=2, G=1, seed=8)
    q = torch.cat([b.q, b.q, b.q])
    out = torch.full_like(q, 7.0)
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    _, lse = paged_attention(q, b.cache, i32(b.indices, gpu), i32([0, 200, 0, 200], gpu), i32([16, 16, 16], gpu), out=out,
                             err=err, return_lse=True)
    b.check(out[:1], lse[:1])
    assert (out[1] == 0).all() and (out[2] == 7).all() and err.item() == 1


def test_hundreds_of_chunks(gpu):
    """Some 580 chunks of a request: a joining wave weighs its share 64 at a time."""
    b = Batch(gpu, [300000], [1], H=1, G=2, D=64, seed=21)
    out, lse = b.run()
    torch.cuda.synchronize()
    b.check(out, lse)


@pytest.mark.parametrize("D,kv,new", [(64, [2000, 700, 5], [60, 41, 1]), (128, [2000, 700, 5], [60, 41, 1]),
                                      (256, [2000, 90], [400, 80])])
def test_many_rows_are_joined(gpu, D, kv, new):
    """2142 and 10080 rows of 21 heads, a count that the rows which a joining wave takes do not divide."""
    b = Batch(gpu, kv, new, H=3, G=7, D=D, seed=22, tree=True)
    out, lse = b.run()
    torch.cuda.synchronize()
    b.check(out, lse)
