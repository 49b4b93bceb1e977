"""norm_rotate, append_paged_kv_cache_rope and append_paged_latent_cache (HIP) at the
ends of their ranges, against the 64-bit oracle: quantised pages of any size, rows
whose squares leave float32's normal numbers, layouts of the outputs, and the sizes
from which on a call takes another kernel."""
import numpy as np
import pytest
import torch

from oracle import mx_oracle as mo
from oracle import rope_oracle as ro
from paceserve_amd.kv_transfer import latent, mx, rope

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
EPS = 1e-6


def f64(x):
    return x.double().cpu().numpy()


def sub_of(dtype):
    return 2.0 ** -25 if dtype is FP16 else 0.0


def rows(rng, shape, dtype, dev, gain=1.0):
    return torch.from_numpy(gain * rng.standard_normal(shape) * np.exp(0.5 * rng.standard_normal(shape[-1]))).to(dtype).to(dev)


def check_turned(got, x, weight, positions, table, interleaved=False, eps=EPS):
    """Rows got [n, heads, D] of x at the positions."""
    g, x, t = f64(got), f64(x), f64(table)
    w = None if weight is None else f64(weight)
    step, sub = torch.finfo(got.dtype).eps, sub_of(got.dtype)
    for i, p in enumerate(positions):
        y, size = ro.turned(x[i], w, eps, t[p], interleaved)
        off, most = np.abs(g[i] - y), ro.bound(y, size, x.shape[-1], step, sub)
        assert (off <= most).all(), f"token {i}: off by {np.max(off / most):.3g} of its bound"


def scale_exponents(amax, fmt):
    """Of blocks' largest magnitudes: the smallest exponents that bring them within the type."""
    with np.errstate(divide="ignore"):
        return np.clip(np.ceil(np.log2(amax / mo.TOP[fmt])), -117, 127)


def check_quantised_keys(data, byte, x, weight, positions, table, interleaved, fmt):
    """Element and scale bytes of keys x [n, heads, D].  The float32 result lies within the
    bound e of y: the scale is that of a block's largest magnitude within e, and rounding
    once adds half a step of the element, at most 2^-4 (2^-2) of the value, or half the
    smallest step."""
    x, t, w = f64(x), f64(table), None if weight is None else f64(weight)
    got = mo.values(data, byte, fmt)
    low, u = (2.0 ** -10, 2.0 ** -4) if fmt == "mxfp8" else (2.0 ** -2, 2.0 ** -2)
    for i, p in enumerate(positions):
        y, size = ro.turned(x[i], w, EPS, t[p], interleaved)
        e = ro.bound(y, size, x.shape[-1], 0.0, 0.0)
        blocks = y.shape[0], -1, mo.BLOCK
        least, most = ((np.abs(y) + s * e).reshape(blocks).max(-1) for s in (-1, 1))
        exponent = byte[i].astype(int) - 127
        assert (exponent >= scale_exponents(np.maximum(least, 0), fmt)).all()
        assert (exponent <= scale_exponents(most, fmt)).all()
        scale = np.repeat(np.exp2(exponent.astype(np.float64)), mo.BLOCK, -1)
        assert (np.abs(got[i] - y) <= np.maximum(u * (np.abs(y) + e), low * scale) + e).all(), f"token {i}"


def append_and_check(gpu, n, Hq, H, D, r, P, dtype, fmt, interleaved, norm=True, tokens=None, seed=0):
    """An append into a cache (fmt None: of the rows' type) whose other slots hold a
    pattern; `tokens`: those looked at (all by default)."""
    rng = np.random.default_rng(seed + n + D)
    pages = -(-n // P) + 3
    table = rope.rotary_table(300, r, device=gpu)
    pos, slots = rng.integers(0, 300, n), rng.permutation(pages * P)[:n]
    slots[rng.integers(0, n, n // 50)] = -1                            # some of them padding
    pos_t = torch.tensor(pos, dtype=torch.int32, device=gpu)
    slot_t = torch.tensor(slots, dtype=torch.int64, device=gpu)
    q, k, v = rows(rng, (n, Hq + 2 * H, D), dtype, gpu).split([Hq, H, H], 1)
    w = rows(rng, (D,), dtype, gpu) if norm else None
    if fmt is None:
        cache = torch.full((pages, 2, P, H, D), 5.0, dtype=dtype, device=gpu)
    else:
        cache = torch.full((pages, 2, P, H, mx.row_width(D, fmt)), 0x35, dtype=torch.uint8, device=gpu)
    was, err = cache.clone(), torch.zeros(1, dtype=torch.int32, device=gpu)
    out = torch.full_like(q, 7.0)
    rope.append_paged_kv_cache_rope(q, k, v, pos_t, slot_t, cache, table, w, w, interleaved=interleaved, out=out, err=err)
    torch.cuda.synchronize()
    assert err.item() == 0
    pad = torch.from_numpy(slots < 0).to(gpu)
    assert (out[pad] == 7).all()
    live = np.flatnonzero(slots >= 0)
    page, at = torch.from_numpy(slots[live] // P).to(gpu), torch.from_numpy(slots[live] % P).to(gpu)
    written = torch.zeros((pages, P), dtype=torch.bool, device=gpu)
    written[page, at] = True
    look = live if tokens is None else np.unique(np.concatenate([live[:3], live[-3:], rng.choice(live, tokens)]))
    li = torch.from_numpy(look).to(gpu)
    lp, la = torch.from_numpy(slots[look] // P).to(gpu), torch.from_numpy(slots[look] % P).to(gpu)
    check_turned(out[li], q[li], w, pos[look], table, interleaved)
    if fmt is None:
        check_turned(cache[lp, 0, la], k[li], w, pos[look], table, interleaved)
        assert torch.equal(cache[page, 1, at], v[torch.from_numpy(live).to(gpu)])
        keep = ~written[:, None, :].expand(-1, 2, -1)
        assert (cache[keep] == 5).all()
        return
    data, byte = mx.elements_and_scales(cache, D)
    for new, old in zip((data, byte), mx.elements_and_scales(was, D)):
        keep = ~written[:, None, :].expand(-1, 2, -1)
        assert torch.equal(new[keep], old[keep])
    codes, c = mo.quantize(f64(v[li]), fmt)                           # values as the quantising append does it
    assert np.array_equal(data[lp, 1, la].cpu().numpy(), mo.pack(codes, fmt))
    assert np.array_equal(byte[lp, 1, la].cpu().numpy(), c)
    check_quantised_keys(data[lp, 0, la].cpu().numpy(), byte[lp, 0, la].cpu().numpy(), k[li], w, pos[look], table,
                         interleaved, fmt)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("H,D,r,P", [(1, 64, 64, 1), (2, 64, 64, 1), (3, 64, 64, 1), (1, 128, 128, 1), (2, 128, 64, 1),
                                     (3, 128, 128, 1), (1, 192, 64, 1), (3, 256, 256, 1), (1, 64, 64, 3), (1, 64, 64, 7)])
def test_quantised_pages_of_any_size(gpu, H, D, r, P, dtype, fmt, interleaved):
    """Halves of 34 and 66 bytes and their multiples, of which few are multiples of 16."""
    append_and_check(gpu, 45, 2 * H, H, D, r, P, dtype, fmt, interleaved)


@pytest.mark.parametrize("eps", [0.0, 2.0 ** -133, 2.0 ** -100])
@pytest.mark.parametrize("power", [-20, -45, -62, -66, -70, -90, -126, -131])
def test_rows_whose_squares_are_below_the_normal_numbers(gpu, power, eps):
    """Rows of 2^power: their mean square is a subnormal number of float32 or less, and counts
    where eps does not hide it.  Beside them rows of ordinary numbers."""
    rng = np.random.default_rng(-power)
    table = rope.rotary_table(8, 64, device=gpu)
    pos = np.array([1, 2, 7])
    at = torch.tensor(pos, dtype=torch.int32, device=gpu)
    q, k = rows(rng, (3, 5, 128), torch.float64, gpu), rows(rng, (3, 2, 64), torch.float64, gpu)
    q[1] *= 2.0 ** power
    q[2, 3] *= 2.0 ** power
    q, k = q.to(BF16), k.to(BF16)
    w, w64 = rows(rng, (128,), BF16, gpu), rows(rng, (64,), BF16, gpu)
    got, _ = rope.norm_rotate(q, None, at, table, w, eps=eps)
    check_turned(got, q, w, pos, table, eps=eps)
    # into a latent cache
    x = rows(rng, (3, 256), torch.float64, gpu)
    x[1:] *= 2.0 ** power
    x = x.to(BF16)
    cache, w = latent.empty_cache(1, 4, 256, device=gpu), rows(rng, (256,), BF16, gpu)
    latent.append_paged_latent_cache(x, k[:, 0], at, torch.arange(3, device=gpu), cache, table, w, eps=eps)
    y, g = f64(x), f64(cache[0, :3, :256])
    y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * f64(w)
    assert (np.abs(g - y) <= ro.bound(y, np.abs(y), 256, torch.finfo(BF16).eps, 0.0)).all()
    # and keys on their way into pages
    kv = torch.zeros((1, 2, 16, 2, 64), dtype=BF16, device=gpu)
    small = (k.double() * 2.0 ** power).to(BF16)
    rope.append_paged_kv_cache_rope(small, small, k, at, torch.arange(3, device=gpu), kv, table, None, w64, eps=eps)
    check_turned(kv[0, 0, :3], small, w64, pos, table, eps=eps)


def test_outputs_in_any_layout_whose_rows_are_apart(gpu):
    """Heads before tokens, rows between other rows, tokens and heads whose rows alternate."""
    rng = np.random.default_rng(3)
    n, H, D = 6, 4, 64
    table = rope.rotary_table(20, 64, device=gpu)
    pos = rng.integers(0, 20, n)
    at = torch.tensor(pos, dtype=torch.int32, device=gpu)
    q = rows(rng, (n, H, D), BF16, gpu)
    want, _ = rope.norm_rotate(q, None, at, table)
    room = torch.zeros(4096, dtype=BF16, device=gpu)
    for strides in ((64, n * 64, 1), (512, 128, 1), (128, 1024, 1), (64 * 8, 64, 1), (64 * 5, 64 * 2, 1)):
        room.zero_()
        got, _ = rope.norm_rotate(q, None, at, table, out_q=room.as_strided((n, H, D), strides))
        assert torch.equal(got, want)
        assert (room != 0).sum() == (want != 0).sum()
    for strides in ((64, 64, 1), (64 * 3, 64, 1), (64 * 2, 64 * 3, 1), (96, 64, 1), (64, 96, 1), (64 * 5 - 32, 64 * 2, 1)):
        with pytest.raises(RuntimeError, match="overlap"):
            rope.norm_rotate(q, None, at, table, out_q=room.as_strided((n, H, D), strides))


def check_every_token(got, x, w, positions, table, interleaved):
    """check_turned in torch's float64, some thousand tokens at a time; the first and the
    last by the oracle."""
    n, _, D = x.shape
    ends = np.array([0, 1, n - 2, n - 1])
    check_turned(got[ends], x[ends], w, positions[ends], table, interleaved)
    r = table.shape[1]
    j = torch.arange(r // 2, device=x.device)
    a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + r // 2)
    for i in range(0, n, 4000):
        y = x[i:i + 4000].double()
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS) * w.double()
        c, s = table[torch.from_numpy(positions[i:i + 4000]).to(x.device)].double()[:, None].split(r // 2, -1)
        size, p, q = y.abs(), y[..., a], y[..., b]
        y[..., a], y[..., b] = p * c - q * s, q * c + p * s
        size[..., a], size[..., b] = (p * c).abs() + (q * s).abs(), (q * c).abs() + (p * s).abs()
        e = (D / 2 + 10) * 2.0 ** -24 * size                          # as the oracle's bound
        most = torch.finfo(x.dtype).eps / 2 * (y.abs() + e) + e + sub_of(x.dtype)
        assert ((got[i:i + 4000].double() - y).abs() <= most).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n,Hq,H,D,r", [(16400, 16, 4, 128, 128), (16385, 8, 4, 128, 64), (9001, 32, 16, 128, 128),
                                        (2100, 40, 30, 256, 256), (20000, 1, 0, 80, 80)])
def test_waves_of_several_turns_and_streamed_rows(gpu, n, Hq, H, D, r, dtype, interleaved):
    """Tokens enough that a wave takes a token's heads in turns, in calls on both sides of the
    64 MiB from which on rows are loaded nontemporally; in place too."""
    rng = np.random.default_rng(n)
    table = rope.rotary_table(300, r, device=gpu)
    pos = rng.integers(0, 300, n)
    at = torch.tensor(pos, dtype=torch.int32, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(n)
    x = torch.randn((n, Hq + H, D), generator=g, device=gpu).to(dtype)
    q, k = x[:, :Hq], x[:, Hq:] if H else None
    w = rows(rng, (D,), dtype, gpu)
    got_q, got_k = rope.norm_rotate(q, k, at, table, w, w if H else None, interleaved=interleaved)
    check_every_token(got_q, q, w, pos, table, interleaved)
    if H:
        check_every_token(got_k, k, w, pos, table, interleaved)
    rope.norm_rotate(q, k, at, table, w, w if H else None, interleaved=interleaved, out_q=q, out_k=k)
    assert torch.equal(q, got_q) and (k is None or torch.equal(k, got_k))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("fmt", [None, "mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n,Hq,H,D,r,P", [(70, 8, 2, 128, 128, 16), (40, 6, 3, 192, 64, 24), (33, 4, 4, 256, 128, 1),
                                          (16400, 8, 2, 128, 128, 16), (9001, 16, 8, 128, 64, 16)])
def test_appends_in_both_pairings_and_many_tokens(gpu, n, Hq, H, D, r, P, dtype, fmt, interleaved):
    append_and_check(gpu, n, Hq, H, D, r, P, dtype, fmt, interleaved, tokens=None if n < 100 else 40)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n,L,P", [(8192, 512, 16), (8193, 512, 24), (8193, 256, 16), (8195, 256, 1), (20001, 512, 64)])
def test_many_latent_rows(gpu, n, L, P, dtype, interleaved):
    """From 8192 rows on a group of lanes takes two, of which the last is alone in an odd call;
    padding and bad slots among them."""
    rng = np.random.default_rng(n + L)
    pages = -(-n // P) + 2
    table = rope.rotary_table(200, 64, device=gpu)
    pos, slots = rng.integers(0, 200, n), rng.permutation(pages * P)[:n]
    slots[rng.integers(0, n, 300)] = -1
    bad = rng.choice(np.flatnonzero(slots[:n - 1] >= 0), 20, replace=False)
    slots[bad[:10]], pos[bad[10:]] = pages * P + 5, 200
    live = slots >= 0
    live[bad] = False
    x, w = rows(rng, (n, L + 64), dtype, gpu), rows(rng, (L,), dtype, gpu)
    where, at = torch.from_numpy(slots[live]).to(gpu), torch.from_numpy(np.flatnonzero(live)).to(gpu)
    for weight in (w, None):
        cache, err = torch.full((pages, P, L + 64), 3.0, dtype=dtype, device=gpu), torch.zeros(1, dtype=torch.int32, device=gpu)
        latent.append_paged_latent_cache(x[:, :L], x[:, L:], torch.tensor(pos, dtype=torch.int32, device=gpu),
                                         torch.tensor(slots, device=gpu), cache, table, weight, interleaved=interleaved,
                                         err=err)
        torch.cuda.synchronize()
        assert err.item() == 20
        flat = cache.view(-1, L + 64)
        got = flat[where]
        look = np.unique(np.concatenate([[0, 1, len(where) - 2, len(where) - 1], rng.integers(0, len(where), 60)]))
        token = np.flatnonzero(live)[look]
        check_turned(got[look][:, None, L:], x[token][:, None, L:], None, pos[token], table, interleaved)
        if weight is None:
            assert torch.equal(got[:, :L], x[at, :L])
        else:
            y, g = f64(x[at, :L]), f64(got[:, :L])
            y = y / np.sqrt((y * y).mean(-1, keepdims=True) + EPS) * f64(w)
            assert (np.abs(g - y) <= ro.bound(y, np.abs(y), L, torch.finfo(dtype).eps, sub_of(dtype))).all()
        rest = torch.ones(pages * P, dtype=torch.bool, device=gpu)
        rest[where] = False
        assert (flat[rest] == 3).all()


@pytest.mark.parametrize("fmt", [None, "mxfp8"])
@pytest.mark.parametrize("n", [5, 9001])
def test_queries_of_an_append_in_place(gpu, n, fmt):
    rng = np.random.default_rng(n)
    table = rope.rotary_table(50, 64, device=gpu)
    at = torch.tensor(rng.integers(0, 50, n), dtype=torch.int32, device=gpu)
    slots = torch.tensor(rng.permutation(n + 11)[:n], device=gpu)
    x, w = rows(rng, (n, 14, 128), BF16, gpu), rows(rng, (128,), BF16, gpu)
    width = 128 if fmt is None else mx.row_width(128, fmt)
    caches = [torch.zeros((n + 11, 2, 1, 2, width), dtype=BF16 if fmt is None else torch.uint8, device=gpu) for _ in range(2)]
    q, k, v = x.split([10, 2, 2], 1)
    kept = x.clone()
    want = rope.append_paged_kv_cache_rope(q, k, v, at, slots, caches[0], table, w, w)
    got = rope.append_paged_kv_cache_rope(q, k, v, at, slots, caches[1], table, w, w, out=q)
    assert got is q and torch.equal(q, want) and torch.equal(x[:, 10:], kept[:, 10:])
    assert torch.equal(caches[0], caches[1])
