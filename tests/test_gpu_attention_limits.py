"""paged_attention (HIP) at the limits of its numbers: values, weights, scores
and caps where the arithmetic could leave the type, and infinities, each
against the 64-bit oracle."""
import math

import numpy as np
import pytest
import torch

from oracle import attention_oracle as ao
from paceserve_amd.kv_transfer.attention import paged_attention
from test_gpu_attention import BF16, FP16, Batch, i32

pytestmark = pytest.mark.gpu


def one_dominant(b, score, key=4.0):
    """Every key zero but the middle token's of each request, whose score is
    `score`; all queries alike."""
    b.q.zero_()
    b.q[:, :, 0] = score * math.sqrt(b.D) / key
    at = []
    for x, n, t in zip(b.rows, b.kv, b.new):
        x[:, 0] = 0
        at.append((n - t) // 2)
        x[at[-1], 0, :, 0] = key
    return at


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T,G,fmt", [(1, 1, None), (20, 1, None), (10, 8, None), (1, 2, "mxfp8"), (10, 8, "mxfp8")])
def test_a_value_at_the_types_limit(gpu, T, G, fmt, D):
    """The row's largest score belongs to a value of 2^127: any weight of more than
    2 on it passes float32, whose largest number is below 2^128."""
    b = Batch(gpu, [700, 90], [T, T], H=1, G=G, D=D, fmt=fmt, seed=T + G)
    for x, at in zip(b.rows, one_dominant(b, 5.0)):
        x[:, 1, :, 3] = 0
        x[at, 1, :, 3] = 2.0 ** 127
        # the block that shares the value's scale: as small a number as it holds is large
        x[at, 1, :, :3] = x[at, 1, :, 4:32] = 0
    b.fill()
    out, lse = b.run()
    torch.cuda.synchronize()
    assert (out[:, :, 3].float() > 1e37).all() and torch.isfinite(out).all()
    b.check(out, lse)


@pytest.mark.parametrize("fmt", [None, "mxfp8", "mxfp4"])
@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("nats", [9, 16, 18, 22])
def test_float16_keeps_many_small_weights(gpu, nats, T, fmt):
    """A dominant token whose value is zero before a long flat tail, whose weights are
    below float16's smallest normal number and whose sum makes the output."""
    b = Batch(gpu, [30000, 200], [T, T], H=1, G=1, D=64, dtype=FP16, fmt=fmt, seed=nats)
    for x, at in zip(b.rows, one_dominant(b, float(nats))):
        x[at, 1] = 0
    b.fill()
    out, lse = b.run()
    torch.cuda.synchronize()
    b.check(out, lse)
    # The bound of check() grants each weight float16's subnormal half step, 2^-25 of
    # the largest weight.  Weights of up to 2^15 leave 2^-40 of it.
    got = out.double().cpu().numpy()
    for r, x in enumerate(b.seen_rows):
        s = slice(b.qo[r], b.qo[r + 1])
        o, l, mean, dots, spread = ao.attend(b.q[s].double().cpu().numpy(), x[:, 0], x[:, 1], 1 / math.sqrt(b.D), 0.0,
                                             ao.visible(len(x), T, None))
        bo, _ = ao.bounds(b.D, torch.finfo(FP16).eps, o, l, mean, dots, spread, 0.0, len(x), 2.0 ** -40)
        # the result is itself rounded to float16, whose subnormals are 2^-24 apart
        assert (np.abs(got[s] - o) <= bo + 2.0 ** -25).all(), \
            f"request {r}: off by {np.max(np.abs(got[s] - o) / (bo + 2.0 ** -25)):.3g} of the bound"


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("kv,T", [([1, 2, 3, 4], 1), ([24, 21], 20), ([9000], 2)])
def test_log_sums_near_zero(gpu, kv, T, dtype):
    """Small scores: a log-sum-exp to a few float32 roundings of its own terms.  Bound: the
    scores' D + 4 roundings of sum |q k|; an exponential's 2^-23 and its argument's 2^-24;
    sums of n / 4 of a lane, then of 4 lanes, and of waves and chunks; the logarithm's 2^-23 of
    itself, at most log2(n); three roundings of the result's terms."""
    b = Batch(gpu, kv, [T] * len(kv), D=64, dtype=dtype, seed=len(kv), q_gain=0.001)
    out, lse = b.run()
    torch.cuda.synchronize()
    for r, x in enumerate(b.seen_rows):
        s = slice(b.qo[r], b.qo[r + 1])
        o, l, mean, dots, spread = ao.attend(b.q[s].double().cpu().numpy(), x[:, 0], x[:, 1], 1 / math.sqrt(b.D), 0.0,
                                             ao.visible(len(x), T, None))
        n, unit = len(x), 2.0 ** -24
        terms = math.log2(n) + dots * math.log2(math.e)
        bound = (b.D + 4) * unit * dots + (3 + min(n, 512) / 4 + (16 if n > 32 else 2)) * unit + 5 * terms * unit
        assert (np.abs(lse[s].double().cpu().numpy() - l) <= bound).all(), \
            f"request {r}: off by {np.max(np.abs(lse[s].double().cpu().numpy() - l) / bound):.3g} of the bound"


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("rising", [False, True])
def test_values_of_float16s_largest_stay_finite(gpu, rising, T):
    """A weighted mean of one value is that value: weights rounded up must not push
    65504 past the type.  Tokens of equal scores have equal roundings."""
    for k in range(24):
        b = Batch(gpu, [600], [T], H=1, G=1, D=64, dtype=FP16, seed=k)
        one_dominant(b, 0.5 + k / 16)
        if rising:                                      # the larger scores come late
            b.rows[0][200:, 0] = 4.0
        b.rows[0][:, 1] = torch.tensor([65504.0, -65504.0] * 32, dtype=torch.float64)
        b.fill()
        out, lse = b.run()
        torch.cuda.synchronize()
        assert torch.isfinite(out).all(), f"score {0.5 + k / 16}"
        b.check(out, lse)


@pytest.mark.parametrize("dtype,fmt", [(BF16, None), (FP16, None), (BF16, "mxfp4")])
@pytest.mark.parametrize("T,G", [(1, 4), (20, 8)])
@pytest.mark.parametrize("cap", [0.25, 3.0, 64.0, 65.0, 1e3, 1e5, 1e6, 1e8, 1e12, 1e30])
def test_soft_caps_of_every_size(gpu, cap, T, G, dtype, fmt):
    """cap * tanh(s / cap): as the cap grows it is s itself."""
    b = Batch(gpu, [500, 70], [T, T], G=G, dtype=dtype, fmt=fmt, seed=T)
    out, lse = b.run(cap)
    torch.cuda.synchronize()
    got, got_l = out.double().cpu().numpy(), lse.double().cpu().numpy()
    for r, x in enumerate(b.seen_rows):
        s = slice(b.qo[r], b.qo[r + 1])
        o, l, mean, dots, spread = ao.attend(b.q[s].double().cpu().numpy(), x[:, 0], x[:, 1], 1 / math.sqrt(b.D), cap,
                                             ao.visible(len(x), T, None))
        # bounds() takes 2^-21 of what it is given for the cap: past 64 a capped score is
        # right to 2^-20 of itself, and it is at most |s| and at most cap
        term = cap if cap <= 64 else 2 * np.minimum(dots, cap)
        bo, bs = ao.bounds(b.D, torch.finfo(dtype).eps, o, l, mean, dots, spread, term, len(x),
                           2.0 ** -25 if dtype is FP16 else 0.0)
        assert (np.abs(got[s] - o) <= bo).all(), f"request {r}: off by {np.max(np.abs(got[s] - o) / bo):.3g} of its bound"
        assert (np.abs(got_l[s] - l) <= bs).all(), f"request {r}: lse off by {np.max(np.abs(got_l[s] - l) / bs):.3g}"


@pytest.mark.parametrize("dtype,fmt", [(BF16, None), (FP16, None), (BF16, "mxfp8")])
@pytest.mark.parametrize("T,G", [(6, 2), (20, 8)])
def test_infinite_values_reach_those_that_see_them(gpu, dtype, fmt, T, G):
    """An infinity makes an output infinite, of its sign, exactly where its token is
    seen; two of opposite signs make it NaN.  (In a quantised cache its block is NaN.)"""
    b = Batch(gpu, [50, 200], [T, T], dtype=dtype, fmt=fmt, tree=True, G=G, seed=3)
    for x, n in zip(b.rows, b.kv):
        x[n - T + 2, 1, 0, 5] = math.inf
        x[n - T + 3, 1, 1, 7] = -math.inf
        x[n - T + 4, 1, 0, 5] = -math.inf
    for r in range(2):
        for i in range(T):
            b.mask[b.qo[r] + i, 0] = np.uint64(1 << i | (4 if i % 3 == 0 else 0) | (8 if i % 2 else 0))
    b.fill()
    out, lse = b.run()
    torch.cuda.synchronize()
    b.check(out, lse)
    got = out.double().cpu().numpy()
    infinite = 0
    for r, x in enumerate(b.seen_rows):
        s = slice(b.qo[r], b.qo[r + 1])
        o = ao.attend(b.q[s].double().cpu().numpy(), x[:, 0], x[:, 1], 1 / math.sqrt(b.D), 0.0,
                      ao.visible(len(x), T, b.mask[s]))[0]
        assert np.array_equal(np.isposinf(got[s]), np.isposinf(o)) and np.array_equal(np.isneginf(got[s]), np.isneginf(o))
        infinite += int(np.isinf(o).sum())
    assert infinite > 0 or fmt is not None


@pytest.mark.parametrize("fmt", [None, "mxfp8"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,G", [(1, 1), (20, 1), (10, 8)])
@pytest.mark.parametrize("size", [10, 12, 13, 14, 15])
def test_scores_far_past_any_exponential(gpu, size, T, G, dtype, fmt):
    """Queries and keys of powers of two, whose scores (up to 2^34) are exact sums: all
    the weight goes to the token with the largest, and the mean of two equal ones."""
    D = 128
    b = Batch(gpu, [700, 90], [T, T], H=1, G=G, D=D, dtype=dtype, fmt=fmt, seed=size)
    b.q.fill_(2.0 ** size)
    want, top = [], []
    for x, n, t in zip(b.rows, b.kv, b.new):
        x[:, 0] = 2.0 ** (size - 1) * torch.where(torch.arange(n) % 3 == 0, 1, -1)[:, None, None]
        for at in (n // 2, n // 5):
            x[at, 0] = 2.0 ** size
            x[at, 0, :, 5] = 2.0 ** (size - 1) * 1.5    # and a sum that is no power of two
        x[:, 1] = torch.round(x[:, 1] * 4).clamp(-6, 6)
        x[n // 5, 1] = x[n // 2, 1] + 2
    b.fill()
    for scale in (None, 0.1, 0.3):
        out, lse = b.run(**({} if scale is None else dict(sm_scale=scale)))
        torch.cuda.synchronize()
        for r, x in enumerate(b.seen_rows):
            n, t, s = len(x), int(b.new[r]), slice(b.qo[r], b.qo[r + 1])
            mean = torch.from_numpy((x[n // 5, 1] + x[n // 2, 1]) / 2).to(gpu)
            assert (out[s].double() - mean).abs().max() <= torch.finfo(dtype).eps * 8, f"scale {scale} request {r}"
            score = (127 * 4.0 ** size + 0.75 * 4.0 ** size) * (scale or 1 / math.sqrt(D))
            # the scale as float32, times log2(e) and back: a few roundings of the score
            assert (lse[s].double() - score - math.log(2)).abs().max() <= 8 * 2.0 ** -24 * score


@pytest.mark.parametrize("T,G,kv", [(1, 1, 100), (1, 4, 9000), (20, 2, 100), (30, 8, 5000)])
@pytest.mark.parametrize("fmt", [None, "mxfp4"])
def test_tokens_on_bad_pages_are_counted(gpu, T, G, kv, fmt):
    """Each token that lies on a page outside the pool once, however many heads, row
    tiles, waves and chunks look at it."""
    b = Batch(gpu, [kv, 90, 64], [T, T, T], G=G, fmt=fmt, seed=4, tree=G == 2)
    b.indices = b.indices.copy()
    last = b.indptr[1] - 1
    b.indices[2], b.indices[last], b.indices[b.indptr[1]] = b.num_pages, 1 << 30, -5
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    out, lse = b.run(err=err)
    torch.cuda.synchronize()
    b.check(out, lse, hidden=lambda r, p: ((p // 16 == 2) | (p // 16 == last)) if r == 0 else (p // 16 == 0) if r == 1
            else p < 0)
    assert err.item() == 32 + (kv - 1) % 16 + 1


def test_lengths_outside_the_pages_are_counted(gpu):
    b = Batch(gpu, [100, 90, 64, 20], [3, 5, 2, 1], seed=4)
    idx, ip, last = b.tables()
    qo = i32(b.qo, gpu)
    want, _ = b.run()
    for at, bad in ((0, 17), (1, -1), (3, 1 << 30), (3, -(1 << 31))):
        err = torch.zeros(1, dtype=torch.int32, device=gpu)
        l2 = last.clone()
        l2[at] = bad
        out = paged_attention(b.q, b.cache, idx, ip, l2, qo, max_q_len=5, err=err)
        assert err.item() == 1
        for r in range(4):
            if r != at:
                assert torch.equal(out[b.qo[r]:b.qo[r + 1]], want[b.qo[r]:b.qo[r + 1]])
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    none = paged_attention(b.q, b.cache, idx, i32([0] * 5, gpu), last, qo, max_q_len=5, err=err)
    assert err.item() == 0 and (none == 0).all()            # without pages the last one's length means nothing
    # offsets past the table: cut to it, and counted
    ip2 = ip.clone()
    ip2[4] += 3
    out = paged_attention(b.q, b.cache, idx, ip2, last, qo, max_q_len=5, err=err)
    assert err.item() == 1 and torch.equal(out, want)
    err.zero_()
    ip2 = ip.clone()
    ip2[0] = -2
    out = paged_attention(b.q, b.cache, idx, ip2, last, qo, max_q_len=5, err=err)
    assert err.item() == 1 and torch.equal(out, want)


def test_requests_past_the_work_items_are_counted(gpu):
    """kv_indptr [0, 200, 0, 200, 0, 200, 200]: pages counted three times over.  The last requests' items lie
    past those that the call has room for: none of them is lost without a count."""
    b = Batch(gpu, [3200, 0, 0, 0, 0, 0], [1, 0, 0, 0, 0, 0], H=2, G=1, seed=8)
    q = b.q.repeat(6, 1, 1)
    out = torch.full_like(q, 7.0)
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    paged_attention(q, b.cache, i32(b.indices, gpu), i32([0, 200, 0, 200, 0, 200, 200], gpu), i32([16] * 6, gpu), out=out,
                    err=err)
    left = [(out[r] == 7).all().item() for r in range(6)]
    assert left[:3] == [False, False, True] and (out[1] == 0).all()
    assert err.item() == sum(left)


def test_a_pool_without_pages(gpu):
    q = torch.randn(3, 8, 64, dtype=BF16, device=gpu)
    for cache in (torch.zeros(0, 2, 16, 2, 64, dtype=BF16, device=gpu),
                  torch.zeros(0, 2, 16, 2, 66, dtype=torch.uint8, device=gpu)):
        idx, err = i32([], gpu), torch.zeros(1, dtype=torch.int32, device=gpu)
        out, lse = paged_attention(q, cache, idx, i32([0] * 4, gpu), i32([0] * 3, gpu), return_lse=True, err=err)
        assert (out == 0).all() and torch.isneginf(lse).all() and err.item() == 0
        # pages named all the same are outside the pool
        out, lse = paged_attention(q, cache, i32([0, 1, 2], gpu), i32([0, 1, 2, 3], gpu), i32([16, 2, 1], gpu),
                                   return_lse=True, err=err)
        assert (out == 0).all() and torch.isneginf(lse).all()


def test_a_split_request_among_many_that_are_not(gpu):
    """Parts are kept for split requests alone: their numbers skip the others'."""
    rng = np.random.default_rng(31)
    kv = rng.integers(1, 60, 600)
    kv[[0, 3, 255, 256, 257, 300, 599]] = [9000, 12000, 0, 9500, 20000, 8800, 15000]
    new = np.minimum(rng.integers(0, 3, 600), kv)
    for H, G in ((1, 2), (4, 4)):
        b = Batch(gpu, kv, new, H=H, G=G, D=64, seed=31)
        out, lse = b.run()
        torch.cuda.synchronize()
        b.check(out, lse)


@pytest.mark.parametrize("dtype,fmt", [(BF16, None), (FP16, "mxfp8")])
def test_prompts_over_the_pages(gpu, dtype, fmt):
    """More than a thousand causal queries of a request, beside a short one and a
    single token, whose row tiles then are as large."""
    b = Batch(gpu, [1500, 700, 40], [1100, 1, 40], H=1, G=2, D=64, dtype=dtype, fmt=fmt, seed=41)
    out, lse = b.run()
    torch.cuda.synchronize()
    b.check(out, lse)
