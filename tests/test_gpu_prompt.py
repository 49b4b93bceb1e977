"""latent_prompt_attention (HIP) against the 64-bit oracle of attention, head by
head; and the expanded form against the absorbed one."""
import math

import numpy as np
import pytest
import torch

from oracle import attention_oracle as ao
from paceserve_amd.kv_transfer.latent import latent_prompt_attention

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


class Prompts:
    def __init__(self, dev, q_len, kv_len, *, heads=2, D=128, dtype=BF16, seed=0, gain=1.5, pad=2):
        rng = np.random.default_rng(seed)
        self.dev, self.dtype, self.heads, self.D = dev, dtype, heads, D
        self.qo, self.ip = (np.concatenate([[0], np.cumsum(x)]) for x in (q_len, kv_len))
        nnz, n = int(self.qo[-1]), int(self.ip[-1])
        self.nnz = nnz

        def rows(*shape):
            return torch.from_numpy(rng.standard_normal(shape)).to(dtype).to(dev)

        self.q = rows(nnz + pad, heads, D + 64) * gain
        kv = rows(n + pad, heads, 2 * D)
        kv[n:] = math.nan                                              # keys of no request
        self.q[nnz:] = math.nan
        self.kv = kv
        self.key, self.value, self.rope = kv[..., :D], kv[..., D:], rows(n + pad, 64)
        self.rope[n:] = math.nan
        self.scale = 1 / math.sqrt(D + 64)

    def run(self, **more):
        args = dict(return_lse=True)
        args.update(more)
        got = latent_prompt_attention(self.q, self.key, self.rope, self.value, i32(self.qo, self.dev),
                                      i32(self.ip, self.dev), **args)
        torch.cuda.synchronize()
        return got

    def check(self, out, lse, causal=True, scale=None, picks=40):
        """All queries of short prompts; of long ones the first, the last and some between."""
        scale = self.scale if scale is None else scale
        rng, eps = np.random.default_rng(1), torch.finfo(self.dtype).eps
        sub = 2.0 ** -25 if self.dtype is FP16 else 0.0
        q, key, value, rope = (x.double().cpu().numpy() for x in (self.q, self.key, self.value, self.rope))
        got_o, got_l = out.double().cpu().numpy(), lse.double().cpu().numpy()
        for b in range(len(self.qo) - 1):
            t, ks = self.qo[b + 1] - self.qo[b], slice(self.ip[b], self.ip[b + 1])
            n = self.ip[b + 1] - self.ip[b]
            at = np.arange(t)
            if t > picks:
                at = np.unique(np.concatenate([[0, 1, t - 2, t - 1], rng.integers(0, t, picks)]))
            sees = (np.arange(n)[None, :] <= (n - t + at)[:, None]) if causal else np.ones((len(at), n), bool)
            for h in range(self.heads):
                keys = np.concatenate([key[ks, h], rope[ks]], 1)
                values = np.concatenate([value[ks, h], np.zeros((n, 64))], 1)
                o, s, mean, dots, spread = ao.attend(q[self.qo[b] + at, h][:, None], keys[:, None],
                                                     np.concatenate([values, np.zeros((n, keys.shape[1] - values.shape[1]))], 1)[:, None],
                                                     scale, 0.0, sees)
                bo, bs = ao.bounds(self.D + 64, eps, o, s, mean, np.abs(dots), spread, 0.0, n, sub)
                o, bo = o[:, 0, :self.D], bo[:, 0, :self.D]
                go, gl = got_o[self.qo[b] + at, h], got_l[self.qo[b] + at, h]
                assert np.array_equal(np.isnan(o), np.isnan(go)), f"request {b} head {h}: NaN in other places"
                fine = np.isfinite(o)
                assert (np.abs(go - o)[fine] <= bo[fine]).all(), \
                    f"request {b} head {h}: out off by {np.max((np.abs(go - o) / bo)[fine]):.3g} of its bound"
                dead = np.isneginf(s[:, 0])
                assert np.array_equal(dead, np.isneginf(gl)) and (go[dead] == 0).all()
                ok = np.isfinite(s[:, 0])
                assert (np.abs(gl - s[:, 0])[ok] <= bs[ok, 0]).all(), f"request {b} head {h}: lse off"


CASES = [
    # queries, keys, heads, D
    ([1], [1], 1, 128),
    ([5, 0, 33, 64], [5, 3, 33, 64], 3, 128),
    ([130, 1, 65], [130, 500, 65], 2, 64),
    ([700], [700], 4, 128),
    ([257, 31], [1000, 31], 2, 128),
    ([3, 2], [2, 0], 2, 64),                                           # queries before the first key see nothing
    ([1] * 40, list(range(1, 41)), 2, 128),
    ([300, 4], [290, 3000], 1, 64),
    ([2049], [2049], 1, 128),
    ([128, 256, 127, 129], [128, 256, 255, 1000], 16, 128),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_matches_the_oracle(gpu, case, dtype, causal):
    q_len, kv_len, heads, D = CASES[case]
    print(f"prompt case {case} {dtype} causal={causal}", flush=True)
    b = Prompts(gpu, q_len, kv_len, heads=heads, D=D, dtype=dtype, seed=case)
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    out = torch.full((b.nnz + 2, heads, D), 7.0, dtype=dtype, device=gpu)
    out, lse = b.run(causal=causal, err=err, out=out)
    b.check(out, lse, causal)
    assert err.item() == 0 and (out[b.nnz:] == 7).all()


def test_slices_and_contiguous_tensors_agree(gpu):
    b = Prompts(gpu, [90, 200], [90, 300], heads=3, seed=1)
    want, lse = b.run()
    b.key, b.value = b.key.contiguous(), b.value.contiguous()
    wide = torch.zeros((b.q.shape[0], 5, 200), dtype=BF16, device=gpu)
    wide[:, 1:4, :192] = b.q
    b.q = wide[:, 1:4, :192]
    room = torch.full((b.q.shape[0], 3, 136), 2.0, dtype=BF16, device=gpu)
    got, again = b.run(out=room[..., :128])
    assert torch.equal(got[:b.nnz], want[:b.nnz]) and torch.equal(again[:b.nnz], lse[:b.nnz]) and (room[..., 128:] == 2).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_what_is_not_seen_cannot_matter(gpu, dtype):
    b = Prompts(gpu, [70, 140], [70, 200], heads=2, dtype=dtype, seed=2)
    key, value = b.kv[..., :128], b.kv[..., 128:]
    value[30, 0, 5], value[31, 1, 6] = math.inf, math.nan
    key[32, 0, 3] = math.nan
    b.rope[70 + 150, 9] = math.nan
    value[70 + 199] = math.nan
    out, lse = b.run()
    b.check(out, lse, picks=10000)
    assert torch.isfinite(out[:30]).all() and torch.isfinite(out[70:70 + 90]).all()


def test_wide_scores_scales_and_large_values(gpu):
    b = Prompts(gpu, [200], [260], heads=2, seed=3, gain=200.0)
    b.check(*b.run())
    for scale in (0.0, -0.2):
        b.check(*b.run(sm_scale=scale), scale=scale)
    b = Prompts(gpu, [100], [100], heads=2, dtype=FP16, seed=4)
    b.value[:] = 65504.0
    out, lse = b.run()
    assert (out[:100] == 65504).all()


def test_bad_requests_are_skipped_and_counted(gpu):
    b = Prompts(gpu, [40, 50, 30], [40, 60, 30], seed=5, pad=0)
    want, _ = b.run()
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    out = torch.full_like(want, 7.0)
    b.run(max_q_len=45, out=out, err=err)
    assert err.item() == 1 and (out[40:90] == 7).all()
    assert torch.equal(out[:40], want[:40]) and torch.equal(out[90:], want[90:])
    ip = b.ip.copy()
    b.ip = np.array([0, 40, 100, 200])                                 # the last request's keys leave the tensor
    err.zero_()
    cut, _ = b.run(err=err)
    assert err.item() == 1 and torch.equal(cut, want)
    b.ip, b.qo = ip, np.array([0, 40, 30, 120])                        # the second runs backwards
    err.zero_()
    out = torch.full_like(want, 7.0)
    b.run(err=err, out=out)
    assert err.item() == 1 and torch.equal(out[:30], want[:30])
    b.qo = np.array([-3, 40, 90, 500])
    err.zero_()
    out = torch.full_like(want, 7.0)
    b.run(err=err, out=out)
    assert err.item() == 2 and torch.equal(out[40:90], want[40:90]) and (out[:40] == 7).all() and (out[90:] == 7).all()


def test_captured_and_on_another_stream(gpu):
    b = Prompts(gpu, [100, 64], [150, 64], heads=4, seed=6, pad=0)
    qo, ip = i32(b.qo, gpu), i32(b.ip, gpu)
    want = latent_prompt_attention(b.q, b.key, b.rope, b.value, qo, ip)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = latent_prompt_attention(b.q, b.key, b.rope, b.value, qo, ip)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = latent_prompt_attention(b.q, b.key, b.rope, b.value, qo, ip, return_lse=True)
    for new, kv in (([100, 64], [150, 64]), ([1, 163], [3, 211]), ([164, 0], [214, 0])):
        b.qo, b.ip = (np.concatenate([[0], np.cumsum(x)]) for x in (new, kv))
        qo.copy_(i32(b.qo, gpu))
        ip.copy_(i32(b.ip, gpu))
        b.q.mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        b.check(out, lse)
        eager, l2 = b.run()
        assert torch.equal(eager, out) and torch.equal(l2, lse)


def test_rows_past_32_bits(gpu):
    """Keys and values behind the first 4 GiB of their tensor."""
    n = 300
    wide = torch.zeros((70000, 128, 256), dtype=BF16, device=gpu)     # 4.6 GB
    b = Prompts(gpu, [n], [n], heads=2, seed=7, pad=0)
    wide[-n:, -2:] = b.kv
    b.key, b.value = wide[:, -2:, :128], wide[:, -2:, 128:]
    rope = torch.zeros((70000, 64), dtype=BF16, device=gpu)
    rope[-n:] = b.rope
    out, lse = latent_prompt_attention(b.q, b.key, rope, b.value, i32([0, n], gpu), i32([70000 - n, 70000], gpu),
                                       return_lse=True)
    torch.cuda.synchronize()
    b.key, b.value = b.kv[..., :128], b.kv[..., 128:]
    b.check(out, lse)


def test_nothing_to_do_and_refusals(gpu):
    b = Prompts(gpu, [4], [4], heads=2, pad=0)
    qo, ip = i32(b.qo, gpu), i32(b.ip, gpu)
    none = latent_prompt_attention(b.q[:0], b.key, b.rope, b.value, i32([0, 0], gpu), ip)
    assert none.shape == (0, 2, 128)
    dead, lse = latent_prompt_attention(b.q, b.key[:0], b.rope[:0], b.value[:0], qo, i32([0, 0], gpu), return_lse=True)
    assert (dead == 0).all() and torch.isneginf(lse).all()
    good = dict(q=b.q, key=b.key, rope_key=b.rope, value=b.value, qo_indptr=qo, kv_indptr=ip)
    for bad in (dict(q=b.q.float()), dict(q=b.q[..., :128]), dict(q=b.q[..., :160]), dict(key=b.key.half()),
                dict(value=b.value[:3]), dict(rope_key=b.rope[:, :32]), dict(key=b.key[..., :64]), dict(qo_indptr=qo[:1]),
                dict(max_q_len=0), dict(sm_scale=math.nan), dict(out=torch.empty_like(b.q)), dict(key=b.key.cpu()),
                dict(key=torch.zeros((4, 2, 129), dtype=BF16, device=gpu)[..., 1:])):
        with pytest.raises((ValueError, RuntimeError)):
            latent_prompt_attention(**{**good, **bad})


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,D", [(1, 128), (2, 64)])
def test_keys_dealt_to_many_workgroups(gpu, heads, D, dtype):
    """Few queries over many keys, one request with fewer keys than there are parts, one
    with none; infinities and NaN in some parts alone."""
    b = Prompts(gpu, [5, 3, 2, 130], [20000, 2, 0, 700], heads=heads, D=D, dtype=dtype, seed=11)
    out, lse = b.run()
    b.check(out, lse)
    assert torch.isneginf(lse[5]).all() and torch.isneginf(lse[8:10]).all()
    wide, _ = b.run(causal=False)
    b.check(*b.run(causal=False), causal=False)
    b.value[50, 0, 5], b.value[15000, heads - 1, 6] = math.inf, -math.inf
    b.value[19998, 0, 7] = math.nan                       # seen by the last two of the five queries
    b.check(*b.run())
    b.value[50, 0, 5] = 0
    b.key[12000, 0, 3] = math.nan
    b.check(*b.run())
    assert torch.isfinite(wide[:10]).all()


def test_more_requests_than_lanes(gpu):
    rng = np.random.default_rng(12)
    q_len = rng.integers(0, 6, 150)
    q_len[[3, 77, 149]] = [200, 129, 300]
    b = Prompts(gpu, q_len, q_len + rng.integers(0, 40, 150), heads=1, seed=12)
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    b.check(*b.run(err=err), picks=8)
    assert err.item() == 0
    want, _ = b.run()
    out = torch.full_like(want, 7.0)
    b.run(max_q_len=150, err=err, out=out)
    long = np.repeat(q_len > 150, q_len)
    assert err.item() == 2 and (out[:b.nnz][long] == 7).all() and torch.equal(out[:b.nnz][~long], want[:b.nnz][~long])


@pytest.mark.parametrize("seed", range(10))
def test_random_prompts(gpu, seed):
    rng = np.random.default_rng(100 + seed)
    batch = int(rng.integers(1, 12))
    q_len = np.where(rng.random(batch) < 0.3, 1, rng.integers(0, 400, batch))
    kv = q_len + np.where(rng.random(batch) < 0.5, 0, rng.integers(0, 900, batch))
    if q_len.sum() == 0:
        q_len[0] = kv[0] = 9
    causal = bool(rng.integers(0, 2))
    print(f"prompts {q_len.tolist()} over {kv.tolist()} causal={causal}", flush=True)
    b = Prompts(gpu, q_len, kv, heads=int(rng.integers(1, 5)), D=[64, 128][seed % 2], dtype=[BF16, FP16][seed // 2 % 2],
                seed=seed)
    b.check(*b.run(causal=causal), causal=causal, picks=12)


@pytest.mark.parametrize("D", [64, 128])
def test_values_at_bfloat16s_largest_exponent(gpu, D):
    """Weighted means of values of 2^127 are finite, also where the keys are dealt out."""
    for q_len, kv_len, heads in (([70, 1], [70, 300], 2), ([5], [20000], 1)):
        b = Prompts(gpu, q_len, kv_len, heads=heads, D=D, seed=13)
        b.value[..., 3] = 2.0 ** 127
        b.value[::3, :, 4] = -2.0 ** 127
        b.value[1::3, :, 4] = 2.0 ** 127
        out, lse = b.run()
        assert torch.isfinite(out[:b.nnz]).all() and (out[:b.nnz, :, 3].float() >= 2.0 ** 126).all()
        b.check(out, lse)
