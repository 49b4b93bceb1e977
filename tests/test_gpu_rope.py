"""norm_rotate, append_paged_kv_cache_rope and append_paged_latent_cache (HIP)
against the 64-bit oracle; every bound is derived from the numbers."""
import math

import numpy as np
import pytest
import torch

from oracle import mx_oracle as mo
from oracle import rope_oracle as ro
from paceserve_amd.kv_transfer import latent, mx, rope

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
EPS = 1e-6


def sub_of(dtype):
    return 2.0 ** -25 if dtype is FP16 else 0.0


def f64(x):
    return x.double().cpu().numpy()


def rows(rng, shape, dtype, dev, gain=1.0):
    return torch.from_numpy(gain * rng.standard_normal(shape) * np.exp(0.5 * rng.standard_normal(shape[-1]))).to(dtype).to(dev)


def check_turned(got, x, weight, positions, table, interleaved, keep=None):
    """Rows got [n, heads, D] of the tokens `keep` (all by default)."""
    g, x, t = f64(got), f64(x), f64(table)
    w = None if weight is None else f64(weight)
    eps, sub = torch.finfo(got.dtype).eps, sub_of(got.dtype)
    for i, p in enumerate(positions):
        if keep is not None and not keep[i]:
            continue
        y, size = ro.turned(x[i], w, EPS, t[p], interleaved)
        off, most = np.abs(g[i] - y), ro.bound(y, size, x.shape[-1], eps, sub)
        assert (off <= most).all(), f"token {i}: off by {np.max(off / most):.3g} of its bound"


SHAPES = [
    # tokens, q heads, kv heads, D, rotary
    (1, 1, 1, 64, 64), (5, 32, 8, 128, 128), (300, 8, 2, 128, 64), (33, 7, 1, 80, 32), (17, 6, 3, 96, 96),
    (40, 4, 4, 192, 96), (9, 16, 2, 256, 256), (3, 2, 1, 1024, 1024), (70, 1, 1, 16, 16), (6000, 2, 1, 64, 32),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_rotate_matches_the_oracle(gpu, shape, dtype, interleaved):
    n, Hq, H, D, r = shape
    rng = np.random.default_rng(n + D)
    table = rope.rotary_table(500, r, device=gpu)
    pos = rng.integers(0, 500, n)
    at = torch.tensor(pos, dtype=torch.int32, device=gpu)
    q, k = rows(rng, (n, Hq, D), dtype, gpu), rows(rng, (n, H, D), dtype, gpu, 3.0)
    wq, wk = rows(rng, (D,), dtype, gpu), rows(rng, (D,), dtype, gpu)
    for a, b in ((wq, wk), (None, None), (wq, None)):
        got_q, got_k = rope.norm_rotate(q, k, at, table, a, b, eps=EPS, interleaved=interleaved)
        torch.cuda.synchronize()
        check_turned(got_q, q, a, pos, table, interleaved)
        check_turned(got_k, k, b, pos, table, interleaved)


def test_slices_in_place_and_without_keys(gpu):
    rng = np.random.default_rng(1)
    table = rope.rotary_table(100, 64, device=gpu)
    pos = rng.integers(0, 100, 50)
    at = torch.tensor(pos, dtype=torch.int32, device=gpu)
    qkv = rows(rng, (50, 12, 128), BF16, gpu)
    was = qkv.clone()
    q, k, _ = qkv.split([8, 2, 2], 1)
    w = rows(rng, (128,), BF16, gpu)
    rope.norm_rotate(q, k, at, table, w, w, out_q=q, out_k=k)
    check_turned(qkv[:, :8], was[:, :8], w, pos, table, False)
    check_turned(qkv[:, 8:10], was[:, 8:10], w, pos, table, False)
    assert torch.equal(qkv[:, 10:], was[:, 10:])
    # the rotated part of each head of a latent model's queries
    x = rows(rng, (50, 3, 192), BF16, gpu)
    was = x.clone()
    got, none = rope.norm_rotate(x[..., 128:], None, at, table, interleaved=True, out_q=x[..., 128:])
    assert none is None and got.data_ptr() == x[..., 128:].data_ptr() and torch.equal(x[..., :128], was[..., :128])
    check_turned(x[..., 128:], was[..., 128:], None, pos, table, True)


def test_positions_outside_the_table_are_counted(gpu):
    rng = np.random.default_rng(2)
    table = rope.rotary_table(10, 64, device=gpu)
    pos = np.array([3, -1, 9, 10, 0, 2 ** 31 - 1])
    at = torch.tensor(pos, dtype=torch.int32, device=gpu)
    q = rows(rng, (6, 40, 64), FP16, gpu)
    out = torch.full_like(q, 7.0)
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    rope.norm_rotate(q, None, at, table, out_q=out, err=err)
    assert err.item() == 3 and (out[[1, 3, 5]] == 7).all()
    check_turned(out, q, None, pos, table, False, keep=(pos >= 0) & (pos < 10))


def test_zero_rows_extremes_and_what_is_not_finite(gpu):
    table = rope.rotary_table(4, 64, device=gpu)
    at = torch.tensor([1, 2, 3, 1], dtype=torch.int32, device=gpu)
    q = torch.zeros((4, 2, 64), dtype=BF16, device=gpu)
    q[1] = 2.0 ** 60
    q[2] = 2.0 ** -70
    q[3, 0] = math.nan
    w = torch.ones(64, dtype=BF16, device=gpu)
    got, _ = rope.norm_rotate(q, None, at, table, w)
    check_turned(got[:3], q[:3], w, [1, 2, 3], table, False)
    assert (got[0] == 0).all() and torch.isnan(got[3, 0]).all() and (got[3, 1] == 0).all()


def test_far_positions_keep_their_angles(gpu):
    """Angles of position 1e6 against arithmetic in 64 bits on the host."""
    table = rope.rotary_table(1000001, 16, device=gpu)
    angle = 1e6 * 10000.0 ** (-np.arange(0, 16, 2) / 16)
    want = np.concatenate([np.cos(angle), np.sin(angle)])
    # 2^-25: rounding; 1e6 * 2^-52 for the angle, with two roundings in its making
    assert np.max(np.abs(f64(table[-1]) - want)) <= 2.0 ** -25 + 4e6 * 2.0 ** -52


def slots_of(rng, n, pages, P):
    return rng.permutation(pages * P)[:n]


@pytest.mark.parametrize("fmt", [None, "mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n,Hq,H,D,r,P", [(1, 4, 1, 64, 64, 16), (70, 8, 2, 128, 128, 16), (40, 6, 3, 192, 64, 24),
                                          (33, 4, 4, 256, 128, 1), (5000, 2, 1, 128, 128, 16)])
def test_rows_in_the_cache(gpu, n, Hq, H, D, r, P, dtype, fmt):
    rng = np.random.default_rng(n + D)
    pages = -(-n // P) + 3
    table = rope.rotary_table(300, r, device=gpu)
    pos, slots = rng.integers(0, 300, n), slots_of(rng, n, pages, P)
    pos_t = torch.tensor(pos, dtype=torch.int32, device=gpu)
    slot_t = torch.tensor(slots, dtype=torch.int64, device=gpu)
    qkv = rows(rng, (n, Hq + 2 * H, D), dtype, gpu)
    q, k, v = qkv.split([Hq, H, H], 1)
    w = rows(rng, (D,), dtype, gpu)
    if fmt is None:
        cache = torch.full((pages, 2, P, H, D), 5.0, dtype=dtype, device=gpu)
    else:
        cache = torch.full((pages, 2, P, H, mx.row_width(D, fmt)), 0x35, dtype=torch.uint8, device=gpu)
    was = cache.clone()
    out = rope.append_paged_kv_cache_rope(q, k, v, pos_t, slot_t, cache, table, w, w)
    torch.cuda.synchronize()
    check_turned(out, q, w, pos, table, False)
    page, at = torch.from_numpy(slots // P).to(gpu), torch.from_numpy(slots % P).to(gpu)
    if fmt is None:
        check_turned(cache[page, 0, at], k, w, pos, table, False)
        assert torch.equal(cache[page, 1, at], v)
        was[page, :, at] = cache[page, :, at]
        assert torch.equal(cache, was)
        return
    data, byte = (x.cpu().numpy() for x in mx.elements_and_scales(cache, D))
    p, s = slots // P, slots % P
    # values are quantised as the quantising append does it
    codes, c = mo.quantize(f64(v), fmt)
    assert np.array_equal(data[p, 1, s], mo.pack(codes, fmt)) and np.array_equal(byte[p, 1, s], c)
    # keys: the float32 result lies within the bound e of y; rounding it once adds half a
    # step of the element, at most 2^-4 (2^-2) of the value, or half the smallest step
    got = mo.values(data[p, 0, s], byte[p, 0, s], fmt)
    low, u = (2.0 ** -10, 2.0 ** -4) if fmt == "mxfp8" else (2.0 ** -2, 2.0 ** -2)
    scale = np.repeat(np.exp2(byte[p, 0, s].astype(np.float64) - 127), 32, -1)
    x, t, wd = f64(k), f64(table), f64(w)
    for i in range(n):
        y, size = ro.turned(x[i], wd, EPS, t[pos[i]], False)
        e = ro.bound(y, size, D, 0.0, 0.0)
        assert (np.abs(got[i] - y) <= np.maximum(u * (np.abs(y) + e), low * scale[i]) + e).all()
        # the scale is that of the block's largest magnitude, or its neighbour where e reaches across a power of two
        top = np.abs(y).reshape(y.shape[0], -1, 32).max(-1)
        most = 448.0 if fmt == "mxfp8" else 6.0
        need = np.clip(np.ceil(np.log2(top / most)), -117, 127)
        assert (np.abs(byte[p, 0, s][i].astype(int) - 127 - need) <= 1).all()
    mask = np.ones((pages, P), bool)
    mask[p, s] = False
    old = mx.elements_and_scales(was, D)
    for new, o in ((data, old[0]), (byte, old[1])):
        assert np.array_equal(new.swapaxes(1, 2)[mask], o.cpu().numpy().swapaxes(1, 2)[mask])


def test_padding_and_bad_slots(gpu):
    rng = np.random.default_rng(5)
    table = rope.rotary_table(20, 64, device=gpu)
    slots = torch.tensor([3, -1, 64, -7, 0, 5, 2 ** 40], dtype=torch.int64, device=gpu)
    pos = torch.tensor([1, -1, 2, 3, 4, 20, 6], dtype=torch.int32, device=gpu)
    q, k, v = (rows(rng, (7, h, 64), BF16, gpu) for h in (4, 1, 1))
    cache = torch.full((4, 2, 16, 1, 64), 9.0, dtype=BF16, device=gpu)
    out = torch.full_like(q, 7.0)
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    rope.append_paged_kv_cache_rope(q, k, v, pos, slots, cache, table, out=out, err=err)
    assert err.item() == 4                                            # three slots and one position
    keep = np.array([1, 0, 0, 0, 1, 0, 0], bool)
    check_turned(out, q, None, [1, 0, 0, 0, 4, 0, 0], table, False, keep=keep)
    assert (out[torch.from_numpy(~keep).to(gpu)] == 7).all()
    assert torch.equal(cache[0, 1, 3], v[0]) and torch.equal(cache[0, 1, 0], v[4]) and (cache == 9).sum().item() == \
        cache.numel() - 4 * 64
    err.zero_()
    lat = latent.empty_cache(4, 16, 256, BF16, gpu)
    c, r = rows(rng, (7, 256), BF16, gpu), rows(rng, (7, 64), BF16, gpu)
    latent.append_paged_latent_cache(c, r, pos, slots, lat, table, err=err)
    assert err.item() == 4 and torch.equal(lat[0, 3, :256], c[0]) and (lat != 0).any(-1).sum().item() == 2


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n,L,P", [(1, 512, 16), (130, 512, 24), (77, 256, 1), (5000, 512, 64)])
def test_latent_rows(gpu, n, L, P, dtype, interleaved):
    rng = np.random.default_rng(n + L)
    pages = -(-n // P) + 2
    table = rope.rotary_table(200, 64, device=gpu)
    pos, slots = rng.integers(0, 200, n), slots_of(rng, n, pages, P)
    x = rows(rng, (n, L + 64), dtype, gpu)
    w = rows(rng, (L,), dtype, gpu)
    for weight in (w, None):
        cache = torch.full((pages, P, L + 64), 3.0, dtype=dtype, device=gpu)
        latent.append_paged_latent_cache(x[:, :L], x[:, L:], torch.tensor(pos, dtype=torch.int32, device=gpu),
                                         torch.tensor(slots, device=gpu), cache, table, weight, interleaved=interleaved)
        torch.cuda.synchronize()
        got = cache.view(-1, L + 64)[torch.from_numpy(slots).to(gpu)]
        check_turned(got[:, None, L:], x[:, None, L:], None, pos, table, interleaved)
        if weight is None:
            assert torch.equal(got[:, :L], x[:, :L])
        else:
            y, g = f64(x[:, :L]), f64(got[:, :L])
            y = y / np.sqrt((y * y).mean(-1, keepdims=True) + EPS) * f64(w)
            assert (np.abs(g - y) <= ro.bound(y, np.abs(y), L, torch.finfo(dtype).eps, sub_of(dtype))).all()
        rest = torch.ones(pages * P, dtype=torch.bool, device=gpu)
        rest[torch.from_numpy(slots).to(gpu)] = False
        assert (cache.view(-1, L + 64)[rest] == 3).all()


def test_slots_past_32_bits(gpu):
    """Rows behind the first 4 GiB of a latent cache and of a KV cache."""
    rng = np.random.default_rng(8)
    table = rope.rotary_table(8, 64, device=gpu)
    pages = 240000                                                    # 4.4 GB of 18 KiB pages
    cache = torch.zeros((pages, 16, 576), dtype=BF16, device=gpu)
    x = rows(rng, (2, 576), BF16, gpu)
    slots = torch.tensor([pages * 16 - 1, 5], device=gpu)
    pos = torch.tensor([3, 4], dtype=torch.int32, device=gpu)
    latent.append_paged_latent_cache(x[:, :512], x[:, 512:], pos, slots, cache, table)
    assert torch.equal(cache[-1, 15, :512], x[0, :512]) and torch.equal(cache[0, 5, :512], x[1, :512])
    check_turned(cache[-1, 15:, None, 512:], x[:1, None, 512:], None, [3], table, False)
    kv = cache.view(-1)[:(1 << 31) + (1 << 20)].view(-1, 2, 16, 1, 64)
    q, k, v = (rows(rng, (1, 1, 64), BF16, gpu) for _ in range(3))
    rope.append_paged_kv_cache_rope(q, k, v, pos[:1], torch.tensor([kv.shape[0] * 16 - 1], device=gpu), kv, table)
    assert torch.equal(kv[-1, 1, 15, 0], v[0, 0])
    check_turned(kv[-1, 0, 15:], k, None, [3], table, False)


def test_captured_and_on_another_stream(gpu):
    rng = np.random.default_rng(9)
    table = rope.rotary_table(64, 128, device=gpu)
    q, k, v = (rows(rng, (12, h, 128), BF16, gpu) for h in (8, 2, 2))
    w = rows(rng, (128,), BF16, gpu)
    pos = torch.zeros(12, dtype=torch.int32, device=gpu)
    slots = torch.zeros(12, dtype=torch.int64, device=gpu)
    cache = torch.zeros((4, 2, 16, 2, 128), dtype=BF16, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rope.append_paged_kv_cache_rope(q, k, v, pos, slots.sub(1), cache, table, w, w)
    torch.cuda.current_stream().wait_stream(side)
    assert (cache == 0).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rope.append_paged_kv_cache_rope(q, k, v, pos, slots, cache, table, w, w)
    for turn in range(3):
        pos.copy_(torch.from_numpy(rng.integers(0, 64, 12)))
        slots.copy_(torch.from_numpy(rng.permutation(64)[:12]))
        k.mul_(-0.5)
        graph.replay()
        torch.cuda.synchronize()
        eager = cache.clone()
        want = rope.append_paged_kv_cache_rope(q, k, v, pos, slots, eager, table, w, w)
        assert torch.equal(out, want) and torch.equal(cache, eager)


def test_nothing_to_do(gpu):
    table = rope.rotary_table(4, 64, device=gpu)
    q = torch.zeros((0, 2, 64), dtype=BF16, device=gpu)
    pos, slots = torch.zeros(0, dtype=torch.int32, device=gpu), torch.zeros(0, dtype=torch.int64, device=gpu)
    a, b = rope.norm_rotate(q, q, pos, table)
    assert a.shape == b.shape == q.shape
    cache = torch.zeros((0, 2, 16, 2, 64), dtype=BF16, device=gpu)
    assert rope.append_paged_kv_cache_rope(q, q, q, pos, slots, cache, table).shape == q.shape
    latent.append_paged_latent_cache(q.view(0, 64).new_zeros((0, 256)), q.view(-1, 64), pos, slots,
                                     latent.empty_cache(1, 16, 256, BF16, gpu), table)


def test_refusals(gpu):
    table = rope.rotary_table(4, 64, device=gpu)
    q, k = torch.zeros((3, 4, 64), dtype=BF16, device=gpu), torch.zeros((3, 2, 64), dtype=BF16, device=gpu)
    pos, slots = torch.zeros(3, dtype=torch.int32, device=gpu), torch.arange(3, device=gpu)
    w = torch.ones(64, dtype=BF16, device=gpu)
    good = dict(q=q, k=k, positions=pos, table=table)
    for bad in (dict(q=q.float()), dict(q=q[0]), dict(k=k.half()), dict(k=k[:2]), dict(k=k[..., :32]),
                dict(positions=pos[:2]), dict(table=table.half()), dict(table=table[:, :24]), dict(q_weight=w.float()),
                dict(q_weight=w[:32]), dict(k=None, k_weight=w), dict(out_q=q[:2]), dict(q=q[..., ::2], k=None),
                dict(table=rope.rotary_table(4, 128, device=gpu)), dict(table=rope.rotary_table(4, 24, device=gpu)),
                dict(eps=-1.0), dict(eps=math.nan), dict(q=torch.zeros((3, 4, 65), dtype=BF16, device=gpu)[..., 1:], k=None)):
        with pytest.raises((ValueError, RuntimeError)):
            rope.norm_rotate(**{**good, **bad})
    cache = torch.zeros((2, 2, 16, 2, 64), dtype=BF16, device=gpu)
    good = dict(query=q, append_key=k, append_value=k, positions=pos, slot_mapping=slots, paged_kv_cache=cache, table=table)
    for bad in (dict(append_key=q), dict(append_value=k.half()), dict(slot_mapping=slots[:2]),
                dict(slot_mapping=slots.float()), dict(paged_kv_cache=cache.half()), dict(paged_kv_cache=cache[0]),
                dict(paged_kv_cache=cache[..., :32]), dict(paged_kv_cache=mx.empty_cache(2, 16, 2, 64, "mxfp8", gpu),
                                                          table=rope.rotary_table(4, 32, device=gpu))):
        with pytest.raises((ValueError, RuntimeError)):
            rope.append_paged_kv_cache_rope(**{**good, **bad})


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_quantised_blocks_that_are_not_finite(gpu, fmt):
    """An infinity or a NaN, given or made by the norm, marks its block of 32 and no other;
    rotated columns spread it to their partner's block."""
    rng = np.random.default_rng(8)
    n, H, D, P = 6, 2, 128, 16
    q, k, v = (rows(rng, (n, H, D), BF16, gpu) for _ in range(3))
    k[1, 0, 5], k[2, 1, 100], v[3, 0, 40], v[4, 1, 127] = math.inf, math.nan, -math.inf, math.nan
    table = rope.rotary_table(50, 64, device=gpu)
    at = torch.arange(n, dtype=torch.int32, device=gpu) + 3
    cache = torch.zeros((2, 2, P, H, mx.row_width(D, fmt)), dtype=torch.uint8, device=gpu)
    rope.append_paged_kv_cache_rope(q, k, v, at, torch.arange(n, device=gpu) + 7, cache, table)
    torch.cuda.synchronize()
    byte = mx.elements_and_scales(cache, D)[1].cpu().numpy()
    marked = np.argwhere(byte == 255).tolist()
    # [page, key or value, place, head, block]
    assert sorted(marked) == sorted([[0, 0, 8, 0, 0], [0, 0, 8, 0, 1], [0, 0, 9, 1, 3], [0, 1, 10, 0, 1], [0, 1, 11, 1, 3]])
