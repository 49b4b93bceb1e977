"""paged_latent_attention (HIP) against the 64-bit oracle of attention: one KV
head, whose keys are the rows and whose values are their latent part.  Bounds
are made from the numbers (oracle.attention_oracle.bounds)."""
import math

import numpy as np
import pytest
import torch

from oracle import attention_oracle as ao
from paceserve_amd.kv_transfer import latent
from paceserve_amd.kv_transfer.latent import paged_latent_attention

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


class Batch:
    """Requests of `kv` tokens whose last `new` are queries, on permuted pages;
    every number that no request's token owns is a NaN."""

    def __init__(self, dev, kv, new, *, heads=4, L=512, P=16, dtype=BF16, tree=False, seed=0, gain=1.0, spare=3):
        rng = self.rng = np.random.default_rng(seed)
        kv, new = np.asarray(kv), np.asarray(new)
        self.dev, self.kv, self.new, self.heads, self.L, self.P, self.dtype = dev, kv, new, heads, L, P, dtype
        pages = -(-kv // P)
        self.num_pages = int(pages.sum()) + spare
        self.indptr = np.concatenate([[0], np.cumsum(pages)])
        self.indices = rng.permutation(self.num_pages)[:self.indptr[-1]]
        self.last = np.where(kv == 0, 0, (kv - 1) % P + 1)
        self.qo = np.concatenate([[0], np.cumsum(new)])
        self.nnz = int(self.qo[-1])
        self.scale = 1 / math.sqrt(L + 64)
        self.rows = [torch.from_numpy(rng.standard_normal((n, L + 64)) * np.exp(0.5 * rng.standard_normal(L + 64)))
                     for n in kv]
        self.q = torch.from_numpy(gain * rng.standard_normal((self.nnz, heads, L + 64))).to(dtype).to(dev)
        self.mask = None
        if tree:
            m = np.zeros((self.nnz, max(1, -(-int(max(new, default=1)) // 64))), np.uint64)
            for b, t in enumerate(new):
                for i in range(t):
                    row = self.qo[b] + i
                    if i:
                        m[row] = m[self.qo[b] + i - 1 - rng.integers(0, min(i, 8))]
                    m[row, i // 64] |= np.uint64(1 << (i % 64))
            self.mask = m
        self.fill()

    def fill(self):
        cache = torch.full((self.num_pages, self.P, self.L + 64), math.nan, dtype=self.dtype)
        self.seen = []
        for b, x in enumerate(self.rows):
            pos = np.arange(len(x))
            page = torch.from_numpy(self.indices[self.indptr[b] + pos // self.P].astype(np.int64))
            cache[page, torch.from_numpy(pos % self.P)] = x.to(self.dtype)
            self.seen.append(x.to(self.dtype).double().numpy())
        self.cache = cache.to(self.dev)

    def tables(self):
        return i32(self.indices, self.dev), i32(self.indptr, self.dev), i32(self.last, self.dev)

    def run(self, **more):
        mask = None if self.mask is None else torch.from_numpy(self.mask.view(np.int64)).to(self.dev)
        args = dict(sm_scale=self.scale, max_q_len=max(1, int(self.new.max())), tree_mask=mask, return_lse=True)
        args.update(more)
        got = paged_latent_attention(self.q, self.cache, *self.tables(), i32(self.qo, self.dev), **args)
        torch.cuda.synchronize()
        return got

    def check(self, out, lse, hidden=None, scale=None):
        scale = self.scale if scale is None else scale
        L, eps = self.L, torch.finfo(self.dtype).eps
        sub = 2.0 ** -25 if self.dtype is FP16 else 0.0
        for b, x in enumerate(self.seen):
            n, t, r = len(x), int(self.new[b]), slice(self.qo[b], self.qo[b + 1])
            if t == 0:
                continue
            sees = ao.visible(n, t, None if self.mask is None else self.mask[r])
            if hidden is not None:
                sees &= ~hidden(b, np.arange(n))[None, :]
            values = np.concatenate([x[:, :L], np.zeros((n, 64))], 1)
            o, s, mean, dots, spread = ao.attend(self.q[r].double().cpu().numpy(), x[:, None], values[:, None], scale, 0.0,
                                                 sees)
            bo, bs = ao.bounds(L + 64, eps, o, s, mean, np.abs(dots), spread, 0.0, n, sub)
            o, bo = o[..., :L], bo[..., :L]
            got_o, got_l = out[r].double().cpu().numpy(), lse[r].double().cpu().numpy()
            assert np.array_equal(np.isnan(o), np.isnan(got_o)), f"request {b}: NaN in other places"
            fine = np.isfinite(o)
            assert np.array_equal(o[~fine & ~np.isnan(o)], got_o[~fine & ~np.isnan(o)])
            assert (np.abs(got_o - o)[fine] <= bo[fine]).all(), \
                f"request {b}: out off by {np.max((np.abs(got_o - o) / bo)[fine]):.3g} of its bound"
            dead = np.isneginf(s)
            assert np.array_equal(dead, np.isneginf(got_l)) and (got_o[dead] == 0).all()
            ok = np.isfinite(s)
            assert (np.abs(got_l - s)[ok] <= bs[ok]).all(), f"request {b}: lse off"


CASES = [
    # kv lengths, queries, heads, latent, page
    ([1], [1], 1, 512, 16),
    ([16, 17, 31, 33, 300], [1] * 5, 16, 512, 16),
    ([700, 33, 5], [1, 1, 1], 8, 256, 16),
    ([513, 64], [1, 1], 128, 512, 16),
    ([40, 9, 130], [5, 9, 2], 5, 512, 24),
    ([100, 64, 63], [33, 64, 1], 1, 256, 1),
    ([300, 70, 40], [3, 2, 1], 32, 512, 64),
    ([5000, 260], [3, 1], 16, 512, 16),
    ([4097], [2], 128, 512, 32),
    ([2100, 40], [7, 5], 9, 256, 16),
    ([0, 20, 0, 7], [0, 4, 0, 0], 3, 512, 16),
    ([257, 300], [70, 3], 3, 512, 7),
    ([90] * 70, [1] * 70, 16, 512, 16),
    ([1500, 20], [1, 1], 100, 256, 16),
    ([333, 333, 1000], [4, 4, 4], 16, 512, 16),
]


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_matches_the_oracle(gpu, case, dtype, tree):
    kv, new, heads, L, P = CASES[case]
    print(f"latent case {case} {dtype} tree={tree}", flush=True)
    b = Batch(gpu, kv, new, heads=heads, L=L, P=P, dtype=dtype, tree=tree, seed=case)
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    b.check(*b.run(err=err))
    assert err.item() == 0


def test_one_token_form_is_the_same(gpu):
    b = Batch(gpu, [300, 1, 17], [1, 1, 1], heads=16)
    out, lse = b.run()
    o2, l2 = paged_latent_attention(b.q, b.cache, *b.tables(), sm_scale=b.scale, return_lse=True)
    assert torch.equal(out, o2) and torch.equal(lse, l2)
    only = paged_latent_attention(b.q, b.cache, *b.tables(), sm_scale=b.scale)
    assert torch.equal(only, out)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,heads", [(6, 2), (6, 4), (20, 3), (20, 6), (20, 16)])
def test_what_is_not_seen_cannot_matter(gpu, T, heads, dtype):
    """Drafted tokens with infinities, NaN and the type's lowest values: rows
    that see them get what the definition gives, the others are untouched."""
    b = Batch(gpu, [50, 200], [T, T], heads=heads, dtype=dtype, tree=True, seed=3, gain=1.5)
    low = float(torch.finfo(dtype).min)
    for x, n in zip(b.rows, b.kv):
        first = n - T
        x[first + 2, 5] = math.inf
        x[first + 3, 520] = math.nan
        x[first + 4, :] = math.nan
        x[first + 5, 300] = low / 4
    for r in range(2):
        for i in range(T):
            b.mask[b.qo[r] + i, 0] = np.uint64((1 << i) | (1 if i % 2 else 0))
    b.fill()
    b.q[:, :, 5] = b.q[:, :, 5].abs() + 0.5               # the infinite score is +inf: a row that sees it is NaN
    b.q[:, :, 300] = 2.0 ** -8 if dtype is FP16 else 2.0 ** -120
    out, lse = b.run()
    b.check(out, lse)
    for r in range(2):
        fine = [i for i in range(T) if i not in (2, 3, 4)]
        assert torch.isfinite(out[[b.qo[r] + i for i in fine]]).all()
        assert torch.isnan(out[b.qo[r] + 2]).any() and torch.isnan(out[b.qo[r] + 3]).all()


def test_infinite_values_reach_those_that_see_them(gpu):
    """A latent of infinities whose scores are finite: its column is infinite for
    every row that sees it, and for no other."""
    b = Batch(gpu, [40, 90], [4, 4], heads=16, tree=True, seed=4)
    for x, n in zip(b.rows, b.kv):
        x[n - 3, 7], x[n - 3, 9] = math.inf, -math.inf
    b.fill()
    b.q[:, :, 7], b.q[:, :, 9] = 0.0, 0.0                  # 0 * inf is NaN: the score of that token is NaN
    out, lse = b.run()
    for r in range(2):
        for i in range(4):
            sees = bool(b.mask[b.qo[r] + i, 0] >> np.uint64(1) & np.uint64(1))
            row = out[b.qo[r] + i]
            assert torch.isnan(row).all() if sees else torch.isfinite(row).all()


def test_rows_that_see_nothing(gpu):
    b = Batch(gpu, [4, 30], [4, 4], heads=16, tree=True, seed=1)
    b.mask[1] = 0                                          # no context and no bit: nothing
    b.mask[5] = 0                                          # a context of 26 tokens
    out, lse = b.run()
    b.check(out, lse)
    assert (out[1] == 0).all() and torch.isneginf(lse[1]).all() and torch.isfinite(lse[5]).all()


def test_fewer_tokens_than_queries(gpu):
    b = Batch(gpu, [3, 40], [5, 2], heads=8, seed=6)
    out, lse = b.run()
    b.check(out, lse)
    assert (out[:2] == 0).all() and torch.isneginf(lse[:2]).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads", [3, 128])
def test_wide_scores_and_scales(gpu, heads, dtype):
    """Scores thousands apart, a scale of zero and a negative one."""
    b = Batch(gpu, [200, 40], [2, 3], heads=heads, seed=2, gain=300.0, dtype=dtype)
    b.check(*b.run())
    for scale in (0.0, -0.1):
        b.check(*b.run(sm_scale=scale), scale=scale)


def test_scores_past_two_to_the_27(gpu):
    """A row's largest weight stays 1 where float32 holds scores in steps of 256."""
    b = Batch(gpu, [64, 700], [1, 2], heads=16, seed=9)
    for x in b.rows:
        x[:, :] = 0.0
        x[:, 0] = 2.0 ** 14
        x[:, 1] = torch.arange(len(x)) % 7 + 1.0
        x[len(x) // 2, 0] = 2.0 ** 14 * 1.0078125
    b.fill()
    b.q[:] = 0
    b.q[:, :, 0] = 2.0 ** 20
    out, lse = b.run()
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    for r in range(2):
        want = b.seen[r][len(b.seen[r]) // 2, :512]
        assert np.array_equal(out[b.qo[r + 1] - 1, 0].double().cpu().numpy(), want)


def test_large_values_stay_finite_in_float16(gpu):
    b = Batch(gpu, [300, 65], [1, 3], heads=5, dtype=FP16, seed=10)
    for x in b.rows:
        x[:, 100:] = 0.0
        x[:, :50], x[:, 50:100] = 65504.0, -65504.0
    b.fill()
    b.q[:, :, :100] = 0.0
    out, lse = b.run()
    assert (out[:, :, :50] == 65504).all() and (out[:, :, 50:100] == -65504).all() and (out[:, :, 100:] == 0).all()
    b.check(out, lse)


@pytest.mark.parametrize("heads", [4, 32, 128])
def test_bad_pages_and_requests_are_skipped_and_counted(gpu, heads):
    b = Batch(gpu, [100, 90, 64], [3, 5, 2], heads=heads, seed=4)
    b.indices = b.indices.copy()
    b.indices[2], b.indices[b.indptr[1]] = b.num_pages, -5        # tokens 32..47 of request 0, 0..15 of request 1
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    out, lse = b.run(err=err)
    b.check(out, lse, hidden=lambda r, p: (p // 16 == 2) if r == 0 else (p // 16 == 0) if r == 1 else p < 0)
    assert err.item() == 32
    b = Batch(gpu, [100, 90, 64], [3, 5, 2], heads=heads, seed=4)
    full, _ = b.run()
    err.zero_()
    out = torch.full_like(full, 7.0)
    b.run(max_q_len=4, out=out, err=err)
    assert err.item() == 1 and (out[3:8] == 7).all()
    b.check(torch.cat([out[:3], full[3:8], out[8:]]), b.run()[1])


def test_rows_behind_the_last_request_are_left(gpu):
    b = Batch(gpu, [100, 90], [3, 5], heads=16, seed=5)
    want, _ = b.run()
    q = torch.cat([b.q, torch.full_like(b.q[:4], math.nan)])
    out = torch.full((12, 16, 512), 5.0, dtype=BF16, device=gpu)
    paged_latent_attention(q, b.cache, *b.tables(), i32(b.qo, gpu), sm_scale=b.scale, max_q_len=5, out=out)
    assert torch.equal(out[:8], want) and (out[8:] == 5).all()


def test_strided_queries_and_output(gpu):
    b = Batch(gpu, [100, 290], [3, 5], heads=6, seed=6)
    want, lse = b.run()
    wide = torch.full((8, 9, 576), math.nan, dtype=BF16, device=gpu)
    wide[:, 2:8] = b.q
    room = torch.full((8, 7, 512), 3.0, dtype=BF16, device=gpu)
    b.q = wide[:, 2:8]
    out, _ = b.run(out=room[:, 1:])
    assert out.data_ptr() == room[:, 1:].data_ptr() and (room[:, 0] == 3).all() and torch.equal(room[:, 1:], want)


@pytest.mark.parametrize("heads", [16, 64, 128])
def test_results_repeat_bit_for_bit(gpu, heads):
    b = Batch(gpu, [6000, 3000], [2, 1], heads=heads, seed=7)
    first = b.run()
    for _ in range(3):
        again = b.run()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    b.check(*first)


def test_a_captured_call_follows_the_tables(gpu):
    """Replays over changed tables, with eager calls and work between them."""
    b = Batch(gpu, [900, 500, 40], [1, 1, 1], heads=16, seed=8)
    idx, ip, last = b.tables()
    room = torch.cat([idx, torch.full((40,), -1, dtype=torch.int32, device=gpu)])
    paged_latent_attention(b.q, b.cache, room, ip, last, sm_scale=b.scale)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = paged_latent_attention(b.q, b.cache, room, ip, last, sm_scale=b.scale, return_lse=True)
    for kv in ([900, 500, 40], [1, 1300, 3], [700, 0, 600], [33, 32, 31]):
        c = Batch(gpu, kv, [1, 1, 1], heads=16, seed=sum(kv), spare=b.num_pages - sum(-(-n // 16) for n in kv))
        b.cache.copy_(c.cache)
        b.q.copy_(c.q)
        room.fill_(-1)
        room[:len(c.indices)] = i32(c.indices, gpu)
        ip.copy_(i32(c.indptr, gpu))
        last.copy_(i32(c.last, gpu))
        graph.replay()
        torch.cuda.synchronize()
        c.check(out, lse)
        eager = paged_latent_attention(b.q, b.cache, room, ip, last, sm_scale=b.scale)
        assert torch.equal(eager, out)


def test_two_streams_at_once(gpu):
    a, b = Batch(gpu, [3000], [2], heads=16, seed=11), Batch(gpu, [2000, 100], [1, 1], heads=16, seed=12)
    want = a.run(), b.run()
    args = [(x.q, x.cache, *x.tables(), i32(x.qo, gpu)) for x in (a, b)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(5):
        for k, x in enumerate((a, b)):
            with torch.cuda.stream(streams[k]):
                got[k].append(paged_latent_attention(*args[k], sm_scale=x.scale, max_q_len=2))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(x, got[k][0]) for x in got[k])
        (a, b)[k].check(got[k][0], want[k][1])


def test_pages_past_4_gib(gpu):
    """The last page of a pool of 4.4 GB."""
    pages = 240000
    b = Batch(gpu, [40], [1], heads=16, seed=13)
    cache = torch.full((pages, 16, 576), math.nan, dtype=BF16, device=gpu)
    where = np.array([pages - 1, 3, pages - 2])
    cache[torch.from_numpy(where).to(gpu)] = b.cache[torch.from_numpy(b.indices.astype(np.int64)).to(gpu)]
    b.cache, b.indices = cache, where
    b.check(*b.run())


@pytest.mark.parametrize("seed", range(12))
def test_random_batches(gpu, seed):
    rng = np.random.default_rng(100 + seed)
    B = int(rng.integers(1, 9))
    new = rng.integers(0, 6, B)
    kv = new + rng.integers(0, [40, 400, 3000][seed % 3], B)
    b = Batch(gpu, kv, new, heads=int(rng.choice([1, 2, 7, 16, 20, 40, 64, 128])), L=int(rng.choice([256, 512])),
              P=int(rng.choice([1, 8, 16, 24, 64])), dtype=[BF16, FP16][seed % 2], tree=bool(rng.integers(0, 2)), seed=seed)
    b.check(*b.run())


def test_refusals(gpu):
    b = Batch(gpu, [20, 20], [1, 1], heads=2)
    idx, ip, last = b.tables()
    good = dict(q=b.q, latent_cache=b.cache, kv_indices=idx, kv_indptr=ip, kv_last_page_len=last, sm_scale=0.1)
    qo, mask = i32([0, 1, 2], gpu), torch.ones((2, 1), dtype=torch.int64, device=gpu)
    for bad in (dict(q=b.q.half()), dict(q=b.q[..., :512]), dict(q=b.q[0]), dict(q=b.q[:, :, ::1].cpu()),
                dict(latent_cache=b.cache[..., :512]), dict(latent_cache=b.cache.float()), dict(latent_cache=b.cache[0]),
                dict(kv_indptr=ip[:2]), dict(q=b.q[:1]), dict(max_q_len=2), dict(qo_indptr=qo),
                dict(qo_indptr=qo[:2], max_q_len=1), dict(qo_indptr=qo, max_q_len=0), dict(sm_scale=math.inf),
                dict(sm_scale=math.nan), dict(tree_mask=mask[:1]), dict(tree_mask=mask.int()),
                dict(out=torch.empty_like(b.q)), dict(out=torch.empty_like(b.q)[..., :512])):
        with pytest.raises((ValueError, RuntimeError)):
            paged_latent_attention(**{**good, **bad})
    with pytest.raises(ValueError):
        latent.empty_cache(1, 16, 128)
    with pytest.raises(ValueError):
        latent.empty_cache(1, 16, 512, torch.float32)


@pytest.mark.parametrize("heads", [1, 32, 128])
def test_values_at_bfloat16s_largest_exponent(gpu, heads):
    """Weighted means of values of 2^127 are finite, over one token or over thousands, in
    one part and joined from several."""
    b = Batch(gpu, [1, 40, 5000], [1, 2, 1], heads=heads, seed=20)
    for x in b.rows:
        x[:, 100] = 2.0 ** 127
        x[:, 101] = 2.0 ** 127 * torch.where(torch.arange(len(x)) % 3 == 0, -1.0, 1.0)
    b.q[..., 100:102] = 0.0
    b.fill()
    out, lse = b.run()
    assert torch.isfinite(out).all() and (out[..., 100].float() >= 2.0 ** 126).all()
    b.check(out, lse)


@pytest.mark.parametrize("heads", [1, 128])
@pytest.mark.parametrize("nats", [9, 16, 18, 22])
def test_float16_keeps_many_small_weights(gpu, nats, heads):
    """One token far above a flat tail of 6000: the tail's weights are small numbers of
    float16, and what they add to the columns in which the first token is zero counts."""
    b = Batch(gpu, [6000], [1], heads=heads, dtype=FP16, seed=21)
    x = b.rows[0]
    x[:] = 0.0
    x[:, 100:164] = torch.from_numpy(b.rng.standard_normal((6000, 64)) * 0.1 + 1.0)
    x[3000, 100:164] = 0.0
    x[3000, 0] = 16.0
    b.q.zero_()
    b.q[..., 0] = nats / 16.0 / b.scale
    b.fill()
    out, lse = b.run()
    b.check(out, lse)
    # weights of 2^(15 - nats / ln 2), more than 2^-17: off by 2^-8 at most, as is the result
    got, p = out[0, 0, 100:164].double().cpu().numpy(), math.exp(-nats)
    want = p * b.seen[0][:, 100:164].sum(0) / (1 + p * 5999)
    assert (np.abs(got - want) <= want * 2.0 ** -7 + 2.0 ** -25).all()
