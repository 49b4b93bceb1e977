"""paged_latent_attention and latent_prompt_attention (HIP) at the ends of their ranges and
where a call's size takes another kernel, against 64 bits; and latent pages through the
channel and ops.move."""
import math
import os
import threading

import numpy as np
import pytest
import torch

from oracle import attention_oracle as ao
from paceserve_amd.kv_transfer import latent, ops
from paceserve_amd.kv_transfer.channel import KVChannel

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


def check_one_above(out, lse, scores, values, dtype):
    """Rows out [..., D] that all see tokens of `scores` (natural units) and `values` [n, D].
    The largest weight is 1, which no type rounds: what the others' rounding moves is half a
    step of what they add (and the sum over all is float32's)."""
    s, v, eps = np.asarray(scores), values.astype(np.float64), torch.finfo(dtype).eps
    p = np.exp(s - s.max())
    want, rest = p @ v / p.sum(), np.delete(p, s.argmax()) @ np.abs(np.delete(v, s.argmax(), 0)) / p.sum()
    # scores of at most 2^5 are off by 2^-19 at most (2^-24 of them in float32, and the scale),
    # weights by as much and by the exponential's 2^-21
    f32 = 2.0 ** -17 * (p @ np.abs(v)) / p.sum()
    bound = eps / 2 * (np.abs(want) + rest) * (1 + eps) + f32 + (2.0 ** -25 if dtype is FP16 else 0.0)
    off = np.abs(out.double().cpu().numpy() - want) / bound
    assert off.max() <= 1, f"off by {off.max():.3g} of its bound"
    total = s.max() + math.log(p.sum())
    assert np.abs(lse.double().cpu().numpy() - total).max() <= 2.0 ** -17 * (1 + abs(total))


@pytest.mark.parametrize("above", [0.12, 1.0037, 2.08298, 2.7, 3.0])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,L", [(1, 512), (16, 256), (32, 512), (20, 256), (128, 512), (40, 256)])
def test_a_token_above_those_before_it_counts_in_full(gpu, heads, L, dtype, above):
    """A first token, many of next to no weight, then one some way above the first: its weight is
    the unit, whatever the maximum was before.  (2.08298 is log 8.0283, nearly midway between
    two of bfloat16's numbers.)  All on one page, which is never cut."""
    rng = np.random.default_rng(heads)
    n, P, at, batch = 100, 128, 70, 3
    rank = np.full(n, -8.0)
    rank[0], rank[at] = 0.0, 1.0
    x = torch.zeros((n, L + 64), dtype=torch.float64)
    x[:, :L] = torch.from_numpy(rng.standard_normal((n, L)))
    x[:, L] = torch.from_numpy(rank)
    x = x.to(dtype)
    cache = latent.empty_cache(1, P, L, dtype, gpu)
    cache.view(-1, L + 64)[:n] = x.to(gpu)
    q = torch.zeros((batch, heads, L + 64), dtype=dtype, device=gpu)
    q[..., L] = 1.0
    out, lse = latent.paged_latent_attention(q, cache, i32([0] * batch, gpu), i32(np.arange(batch + 1), gpu),
                                             i32([n] * batch, gpu), sm_scale=above, return_lse=True)
    torch.cuda.synchronize()
    assert torch.equal(out, out[:1, :1].expand_as(out)) and torch.equal(lse, lse[:1, :1].expand_as(lse))
    check_one_above(out[:2], lse[:2], rank * above, x[:, :L].double().numpy(), dtype)


@pytest.mark.parametrize("above", [0.12, 1.0037, 2.08298, 2.7, 3.0])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
def test_a_key_above_those_before_it_counts_in_full(gpu, D, dtype, above):
    rng = np.random.default_rng(D)
    n, t, at, heads = 300, 150, 70, 500
    assert latent._prompt_workspace_bytes(t, n, 1, heads, D, 0) == 0          # no keys are dealt out
    rank = np.full(n, -8.0)
    rank[0], rank[at] = 0.0, 1.0
    value = torch.from_numpy(rng.standard_normal((n, 1, D))).to(dtype)
    rope = torch.zeros((n, 64), dtype=dtype, device=gpu)
    rope[:, 3] = torch.from_numpy(rank)
    q = torch.zeros((t, heads, D + 64), dtype=dtype, device=gpu)
    q[..., D + 3] = 1.0
    key = torch.zeros((n, 1, D), dtype=dtype, device=gpu)
    out, lse = latent.latent_prompt_attention(q, key.expand(-1, heads, -1), rope, value.to(gpu).expand(-1, heads, -1),
                                              i32([0, t], gpu), i32([0, n], gpu), sm_scale=above, causal=False,
                                              return_lse=True)
    torch.cuda.synchronize()
    assert torch.equal(out, out[:1, :1].expand_as(out)) and torch.equal(lse, lse[:1, :1].expand_as(lse))
    check_one_above(out[:, 0], lse[:, 0], rank * above, value[:, 0].double().numpy(), dtype)


def attend_and_check(gpu, kv, new, heads, L, P, dtype, tree=False, tokens=6, some_heads=6, seed=0):
    """Requests of `kv` tokens whose last `new` are queries; a few tokens and heads of each
    against the oracle (heads share their keys).  Slots that no token owns are NaN."""
    rng = np.random.default_rng(seed)
    kv, new = np.asarray(kv), np.asarray(new)
    pages = -(-kv // P)
    num_pages = int(pages.sum()) + 3
    indptr, qo = (np.concatenate([[0], np.cumsum(x)]) for x in (pages, new))
    indices = rng.permutation(num_pages)[:indptr[-1]].astype(np.int64)
    nnz, scale = int(qo[-1]), 1 / math.sqrt(L + 64)
    cache = torch.full((num_pages, P, L + 64), math.nan, dtype=dtype)
    seen = []
    for b, n in enumerate(kv):
        x = torch.from_numpy(rng.standard_normal((n, L + 64)) * np.exp(0.5 * rng.standard_normal(L + 64))).to(dtype)
        at = np.arange(n)
        cache[indices[indptr[b] + at // P], at % P] = x
        seen.append(x.double().numpy())
    cache = cache.to(gpu)
    g = torch.Generator(device=gpu).manual_seed(seed)
    q = torch.randn((nnz, heads, L + 64), generator=g, device=gpu).to(dtype)
    mask = None
    if tree:
        mask = np.zeros((nnz, -(-int(new.max()) // 64)), np.uint64)
        for b, t in enumerate(new):
            for i in range(t):
                row = qo[b] + i
                if i:
                    mask[row] = mask[row - 1 - rng.integers(0, min(i, 8))]
                mask[row, i // 64] |= np.uint64(1 << (i % 64))
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    out, lse = latent.paged_latent_attention(
        q, cache, i32(indices, gpu), i32(indptr, gpu), i32((kv - 1) % P + 1, gpu), i32(qo, gpu), sm_scale=scale,
        max_q_len=int(new.max()), tree_mask=None if mask is None else torch.from_numpy(mask.view(np.int64)).to(gpu),
        return_lse=True, err=err)
    torch.cuda.synchronize()
    assert err.item() == 0 and torch.isfinite(out).all() and torch.isfinite(lse).all()
    eps, sub = torch.finfo(dtype).eps, 2.0 ** -25 if dtype is FP16 else 0.0
    for b, x in enumerate(seen):
        n, t = len(x), int(new[b])
        i = np.unique(np.concatenate([[0, t - 1], rng.integers(0, t, tokens)]))
        h = np.unique(np.concatenate([[0, heads - 1], rng.integers(0, heads, some_heads)]))
        sees = ao.visible(n, t, None if mask is None else mask[qo[b]:qo[b + 1]])[i]
        at = np.ix_(qo[b] + i, h)
        o, s, mean, dots, spread = ao.attend(q.double().cpu().numpy()[at], x[:, None],
                                             np.concatenate([x[:, :L], np.zeros((n, 64))], 1)[:, None], scale, 0.0, sees)
        bo, bs = ao.bounds(L + 64, eps, o, s, mean, dots, spread, 0.0, n, sub)
        off = np.abs(out.double().cpu().numpy()[at] - o[..., :L]) / bo[..., :L]
        assert (off <= 1).all(), f"request {b}: out off by {off.max():.3g} of its bound"
        assert (np.abs(lse.double().cpu().numpy()[at] - s) <= bs).all(), f"request {b}: lse off"


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("kv,new,heads,L,P", [
    ([5000], [40], 128, 512, 16), ([3000, 2500], [35, 30], 64, 256, 16), ([1300, 90, 2049], [70, 3, 65], 33, 512, 24),
    ([900] * 9, [4] * 9, 128, 256, 64)])
def test_split_calls_of_many_rows(gpu, kv, new, heads, L, P, dtype, tree):
    """4096 query rows and more, whose parts a wave each joins."""
    assert sum(new) * heads >= 4096
    pages = sum(-(-n // P) for n in kv)
    assert latent._workspace_bytes(len(kv), heads, L, max(new), pages, P) > 0
    print(f"latent {kv} {new} {heads} {L} {P} {dtype} {tree}", flush=True)
    attend_and_check(gpu, kv, new, heads, L, P, dtype, tree, tokens=3, some_heads=3)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("L", [256, 512])
@pytest.mark.parametrize("kv,new,heads,P", [
    ([6000], [1], 20, 16), ([6000], [1], 32, 16), ([33, 300, 1, 64], [1] * 4, 17, 24), ([4097, 40], [3, 2], 10, 16),
    ([130, 700, 31], [2, 2, 1], 16, 1), ([2000] * 12, [4] * 12, 8, 64), ([5000, 6000], [30, 31], 1, 7)])
def test_two_tiles_of_rows(gpu, kv, new, heads, P, L, dtype, tree):
    """17 to 32 query rows a request: two tiles, of which the second is part empty; requests
    whole and cut into chunks, in both widths."""
    print(f"latent {kv} {new} {heads} {L} {P} {dtype} {tree}", flush=True)
    attend_and_check(gpu, kv, new, heads, L, P, dtype, tree, tokens=2, some_heads=4)


@pytest.mark.parametrize("P,L,dtype", [(16, 512, BF16), (5, 256, FP16), (1, 512, BF16)])
def test_latent_pages_through_the_channel_and_move(gpu, P, L, dtype):
    rng = np.random.default_rng(P)
    layers, num, n = 3, 40, 17
    src = [torch.from_numpy(rng.standard_normal((num, P, L + 64))).to(dtype).to(gpu) for _ in range(layers)]
    s_ids, d_ids = rng.permutation(num)[:n].tolist(), rng.permutation(num)[:n].tolist()

    def check(dst):
        torch.cuda.synchronize()
        rest = sorted(set(range(num)) - set(d_ids))
        for a, b in zip(dst, src):
            assert torch.equal(a[d_ids].view(torch.int16), b[s_ids].view(torch.int16)) and (a[rest] == 7).all()

    dst = [torch.full_like(x, 7.0) for x in src]
    ops.move(src, s_ids, dst, d_ids)
    check(dst)
    dst = [torch.full_like(x, 7.0) for x in src]
    name = f"pace_latent_test_{os.getpid()}_{P}"
    rx = KVChannel.create(name, 1 << 20, 4)
    tx = KVChannel.open(name, timeout=10)
    failed = []

    def sender():
        try:
            tx.send(src, s_ids, b"rows", timeout=30)
        except Exception as e:                                         # reported below
            failed.append(repr(e))

    thread = threading.Thread(target=sender)
    thread.start()
    try:
        h = rx.recv_header(timeout=30)
        assert (h.meta, h.num_layers, h.n_pages, h.page_bytes) == (b"rows", layers, n, P * (L + 64) * 2)
        rx.recv(dst, d_ids, timeout=30)
        check(dst)
    finally:
        thread.join(timeout=60)
        tx.close()
        rx.close()
    assert not failed, failed


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("q_len,kv_len,heads,D", [([2049], [2049], 50, 128), ([130, 700], [600, 700], 130, 64),
                                                  ([2300], [3000], 50, 64), ([511] * 8, [600] * 8, 26, 128)])
def test_prompts_of_four_workgroups_a_cu(gpu, q_len, kv_len, heads, D, dtype, causal):
    """769 to 1024 workgroups, of which two at a time run on a CU instead of three."""
    tiles = -(-sum(q_len) // 128) + (len(q_len) - 1) // 2
    assert 768 < tiles * heads <= 1024
    nnz, n, scale = sum(q_len), sum(kv_len), 1 / math.sqrt(D + 64)
    assert latent._prompt_workspace_bytes(nnz, n, len(q_len), heads, D, int(causal)) == 0
    rng = np.random.default_rng(nnz)
    g = torch.Generator(device=gpu).manual_seed(nnz)
    q = (1.5 * torch.randn((nnz, heads, D + 64), generator=g, device=gpu)).to(dtype)
    kv = torch.randn((n, heads, 2 * D), generator=g, device=gpu).to(dtype)
    rope = torch.randn((n, 64), generator=g, device=gpu).to(dtype)
    qo, ip = (np.concatenate([[0], np.cumsum(x)]) for x in (q_len, kv_len))
    out, lse = latent.latent_prompt_attention(q, kv[..., :D], rope, kv[..., D:], i32(qo, gpu), i32(ip, gpu), causal=causal,
                                              return_lse=True)
    torch.cuda.synchronize()
    eps, sub = torch.finfo(dtype).eps, 2.0 ** -25 if dtype is FP16 else 0.0
    for b, (t, m) in enumerate(zip(q_len, kv_len)):
        at = np.unique(np.concatenate([[0, t - 1], rng.integers(0, t, 6)]))
        sees = (np.arange(m)[None, :] <= (m - t + at)[:, None]) if causal else np.ones((len(at), m), bool)
        for h in (0, int(rng.integers(1, heads - 1)), heads - 1):
            key = torch.cat([kv[ip[b]:ip[b + 1], h, :D], rope[ip[b]:ip[b + 1]]], 1).double().cpu().numpy()
            value = np.concatenate([kv[ip[b]:ip[b + 1], h, D:].double().cpu().numpy(), np.zeros((m, 64))], 1)
            o, s, mean, dots, spread = ao.attend(q[qo[b] + at, h].double().cpu().numpy()[:, None], key[:, None], value[:, None],
                                                 scale, 0.0, sees)
            bo, bs = ao.bounds(D + 64, eps, o, s, mean, dots, spread, 0.0, m, sub)
            got, sums = (x[qo[b] + at, h].double().cpu().numpy() for x in (out, lse))
            assert (np.abs(got - o[:, 0, :D]) <= bo[:, 0, :D]).all() and (np.abs(sums - s[:, 0]) <= bs[:, 0]).all()
