"""Appends into a quantised cache and page conversion (HIP) against the 64-bit
oracle, byte for byte: every element and scale is exact by definition, so
nothing here has a tolerance."""
import numpy as np
import pytest
import torch

from oracle import kv_oracle as orc
from oracle import mx_oracle as mo
from paceserve_amd.kv_transfer import append as ap
from paceserve_amd.kv_transfer import mx, ops
from paceserve_amd.kv_transfer.swap import SwapSpace

pytestmark = pytest.mark.gpu
FORMATS = ["mxfp8", "mxfp4"]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


def mixed(shape, dtype, rng, dev):
    """Values of every kind: normal ones at scales from 2^-20 to 2^20 (within
    the type), raw bit patterns (infinities, NaN, subnormals), zeros, and blocks
    whose largest magnitude lies at a scale's border."""
    n = int(np.prod(shape)) // 32
    x = torch.from_numpy(rng.standard_normal((n, 32)) * 2.0 ** rng.integers(-20, 12, (n, 1))).to(dtype)
    kind = rng.integers(0, 8, n)
    bits = {2: torch.int16, 4: torch.int32}[x.element_size()]
    raw = torch.from_numpy(rng.integers(-2 ** (8 * x.element_size() - 1), 2 ** (8 * x.element_size() - 1), (n, 32)))
    x[kind == 0] = raw.to(bits).view(dtype)[kind == 0]
    x[kind == 1] = 0
    top = torch.from_numpy(np.array([448, 450, 6, 6.125, 7, 224, 3.0])[rng.integers(0, 7, n)])
    x[:, 3] = torch.where(torch.from_numpy(kind == 2), top.to(dtype), x[:, 3])
    x[kind == 3] = torch.finfo(dtype).max * torch.from_numpy(rng.choice([-1.0, 1.0, 0.5], (n, 32)))[kind == 3].to(dtype)
    return x.reshape(shape).to(dev)


def f64(t):
    return t.double().cpu().numpy()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,D,P,R,strided", [
    (8, 128, 16, 6, True), (1, 64, 16, 5, False), (2, 32, 24, 70, True), (4, 128, 16, 130, False),
    (5, 96, 16, 4, False), (1, 32, 16, 300, False), (3, 256, 7 * 16, 3, True), (32, 128, 1, 4, False)])
def test_append_matches_the_oracle(gpu, dtype, fmt, H, D, P, R, strided):
    print(f"append_mx {dtype} {fmt} H={H} D={D} P={P} R={R} strided={strided}", flush=True)
    rng = np.random.default_rng(H * D + P + R)
    prior, app = rng.integers(0, 40, R), rng.integers(1, 25, R)
    app[::2] = 1
    if R > 6:
        app[3::7] = 0
    total = prior + app
    pages = -(-total // P)
    NP = int(pages.sum()) + 5
    kv_indptr = np.concatenate([[0], np.cumsum(pages)])
    kv_indices = rng.permutation(NP)[: kv_indptr[-1]]
    last = np.where(total % P == 0, P, total % P)
    append_indptr = np.concatenate([[0], np.cumsum(app)])
    nnz = int(append_indptr[-1])
    if strided:
        qkv = mixed((nnz, 4 * H, D), dtype, rng, gpu)
        k, v = qkv[:, H:2 * H], qkv[:, 3 * H:]
    else:
        k, v = mixed((nnz, H, D), dtype, rng, gpu), mixed((nnz, H, D), dtype, rng, gpu)
    width = mx.row_width(D, fmt)
    cache = torch.from_numpy(rng.integers(0, 256, (NP, 2, P, H, width), dtype=np.uint8)).to(gpu)
    want = cache.cpu().numpy().copy()
    seq = orc.get_seq_lens(kv_indptr, last, P)
    bi, pos = orc.get_batch_indices_positions(append_indptr, seq, nnz)
    data, byte = mo.split(want, D)
    data, byte = data.copy(), byte.copy()
    page, slot = kv_indices[kv_indptr[bi] + pos // P], pos % P
    for half, x in ((0, k), (1, v)):
        codes, b = mo.quantize(f64(x), fmt)
        data[page, half, slot], byte[page, half, slot] = mo.pack(codes, fmt), b
    want = np.concatenate([data.reshape(NP, 2, -1), byte.reshape(NP, 2, -1)], -1).reshape(want.shape)
    fused, err = cache.clone(), torch.zeros(1, dtype=torch.int32, device=gpu)
    tables = i32(kv_indices, gpu), i32(kv_indptr, gpu), i32(last, gpu)
    mx.append_paged_kv_cache_mx(k, v, i32(bi, gpu), i32(pos, gpu), cache, *tables, err=err)
    mx.append_paged_kv_cache_mx_indptr(k, v, i32(append_indptr, gpu), fused, *tables, err=err)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(cache.cpu().numpy(), want)
    np.testing.assert_array_equal(fused.cpu().numpy(), want)
    assert err.item() == 0


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_skips_and_counts_what_is_out_of_range(gpu, fmt):
    D = 64
    cache = torch.zeros(4, 2, 8, 1, mx.row_width(D, fmt), dtype=torch.uint8, device=gpu)
    k = torch.ones(5, 1, D, dtype=torch.float16, device=gpu)
    kv_indptr, kv_indices = i32([0, 1, 2], gpu), i32([3, 7], gpu)          # page 7 does not exist
    bi, pos = i32([0, 1, 5, 0, -1], gpu), i32([1, 0, 0, 8, 0], gpu)        # no request 5 or -1, no second page
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    mx.append_paged_kv_cache_mx(k, k, bi, pos, cache, kv_indices, kv_indptr, i32([2, 1], gpu), err=err)
    e, s = mx.elements_and_scales(cache, D)
    assert err.item() == 4
    assert (e[3, :, 1] != 0).all() and (s[3, :, 1] != 0).all()
    assert int((cache != 0).sum()) == 2 * mx.row_width(D, fmt)
    err.zero_()
    cache.zero_()
    # the fused form: request 0's two tokens start before position 0, request 1's page is past the pool
    mx.append_paged_kv_cache_mx_indptr(k, k, i32([0, 2, 4], gpu), cache, kv_indices, kv_indptr, i32([1, 2], gpu),
                                       err=err)
    assert err.item() == 4 and int((cache != 0).sum()) == 2 * mx.row_width(D, fmt)


def pools(L, N, P, H, D, fmt, dtype, rng, dev):
    plain = [mixed((N, 2, P, H, D), dtype, rng, dev) for _ in range(L)]
    small = [torch.from_numpy(rng.integers(0, 256, (N, 2, P, H, mx.row_width(D, fmt)), dtype=np.uint8)).to(dev)
             for _ in range(L)]
    return plain, small


@pytest.mark.parametrize("bad", [False, True])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L,n,P,H,D", [(2, 9, 16, 8, 128), (3, 5, 16, 1, 32), (1, 1, 16, 1, 64), (70, 3, 16, 1, 64),
                                       (2, 130, 24, 4, 96), (1, 7, 16, 5, 256)])
def test_pages_convert_both_ways(gpu, dtype, fmt, L, n, P, H, D, bad):
    print(f"pages {dtype} {fmt} L={L} n={n} P={P} H={H} D={D} bad={bad}", flush=True)
    rng = np.random.default_rng(L * n * D)
    N = n + 4
    plain, small = pools(L, N, P, H, D, fmt, dtype, rng, gpu)
    s_ids, d_ids = rng.permutation(N)[:n], rng.permutation(N)[:n]
    if bad:
        s_ids[n // 2], d_ids[n - 1] = N, -1
    ok = [j for j in range(n) if 0 <= s_ids[j] < N and 0 <= d_ids[j] < N]
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    want = [t.cpu().numpy().copy() for t in small]
    for l in range(L):
        for j in ok:
            for half in (0, 1):
                want[l][d_ids[j], half] = mo.page_half(f64(plain[l][s_ids[j], half]), fmt).reshape(want[l].shape[2:])
    mx.quantize_pages(plain, i32(s_ids, gpu), small, i32(d_ids, gpu), err=err)
    for l in range(L):
        np.testing.assert_array_equal(small[l].cpu().numpy(), want[l])
    assert err.item() == L * (n - len(ok))
    # and back, to other pages of a pool with other contents
    back = [mixed((N, 2, P, H, D), dtype, rng, gpu) for _ in range(L)]
    old = [t.clone() for t in back]
    b_ids = rng.permutation(N)[:n]
    data, byte = mo.split(np.stack(want), D)
    with np.errstate(over="ignore"):
        vals = torch.from_numpy(mo.values(data, byte, fmt)).to(dtype)
    err.zero_()
    mx.dequantize_pages(small, i32(d_ids, gpu), back, i32(b_ids, gpu), err=err)
    for l in range(L):
        for j in range(n):
            if 0 <= d_ids[j] < N:
                old[l][b_ids[j]] = vals[l, d_ids[j]].to(gpu)
        assert torch.equal(torch.isnan(back[l]), torch.isnan(old[l]))
        assert torch.equal(torch.nan_to_num(back[l], 0, 9e4, -9e4), torch.nan_to_num(old[l], 0, 9e4, -9e4))
    assert err.item() == (L if bad else 0)


def test_layer_ranges_and_host_ids(gpu):
    rng = np.random.default_rng(3)
    plain, small = pools(5, 6, 16, 2, 64, "mxfp8", torch.bfloat16, rng, gpu)
    before = [t.clone() for t in small]
    mx.quantize_pages(plain, [4, 0], small, [1, 5], layer_begin=1, layer_end=3)
    for l in range(5):
        same = [bool((small[l][i] == before[l][i]).all()) for i in range(6)]
        assert same == [True] * 6 if l not in (1, 2) else same == [True, False, True, True, True, False]
    with pytest.raises(ValueError, match="more than once"):
        mx.quantize_pages(plain, [4, 0], small, [1, 1])
    with pytest.raises(ValueError, match="source ids but"):
        mx.quantize_pages(plain, [4, 0], small, [1])
    with pytest.raises(ValueError, match="no format"):
        mx.quantize_pages([t[..., :32].contiguous() for t in plain], [0], small, [1])
    with pytest.raises(ValueError, match="differ in page size"):
        mx.quantize_pages([t[:, :, :8].contiguous() for t in plain], [0], small, [1])
    with pytest.raises(ValueError, match="uint8"):
        mx.dequantize_pages(plain, [0], plain, [1])
    with pytest.raises(ValueError, match="is converted"):
        mx.quantize_pages(small, [0], small, [1])
    mx.quantize_pages(plain, [], small, [])
    # half a quantised page is no multiple of 16 bytes: 24 * 3 * 96 * 33 / 32 = 7128
    odd, odd_small = pools(2, 6, 24, 3, 96, "mxfp8", torch.bfloat16, rng, gpu)
    with pytest.raises(RuntimeError, match="multiple of 16 bytes"):
        mx.quantize_pages(odd, [0], odd_small, [1])


def test_append_refuses_in_python(gpu):
    cache = mx.empty_cache(4, 16, 2, 64, "mxfp8", gpu)
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=gpu)
    ip, idx, last = i32([0, 1], gpu), i32([0], gpu), i32([3], gpu)
    ai = i32([0, 3], gpu)
    for bad_k, msg in ((k.to(torch.float8_e4m3fn), "bfloat16"), (k[:, :1], "must be"), (k.transpose(0, 1), "must be"),
                       (k[:, :, :32], "contiguous"), (torch.zeros(3, 2, 96, dtype=torch.bfloat16, device=gpu), "no f"),
                       (k[:2], "differ"), (k.float(), "differ")):
        v = k if msg == "differ" else bad_k
        with pytest.raises(ValueError, match=msg):
            mx.append_paged_kv_cache_mx_indptr(bad_k, v, ai, cache, idx, ip, last)
    with pytest.raises(ValueError, match="kv_indptr needs"):
        mx.append_paged_kv_cache_mx_indptr(k, k, i32([0, 1, 3], gpu), cache, idx, ip, last)
    with pytest.raises(ValueError, match="one entry per"):
        mx.append_paged_kv_cache_mx(k, k, i32([0], gpu), i32([0], gpu), cache, idx, ip, last)
    with pytest.raises(ValueError, match="uint8 device tensor"):
        mx.append_paged_kv_cache_mx_indptr(k, k, ai, cache[:, :, :8], idx, ip, last)


def test_side_stream_and_graph_replays(gpu):
    """An append and both conversions captured together, replayed over new rows
    with eager work between, against the eager calls."""
    rng = np.random.default_rng(8)
    plain, small = pools(2, 6, 16, 2, 128, "mxfp8", torch.bfloat16, rng, gpu)
    back = [torch.zeros_like(t) for t in plain]
    k, v = mixed((5, 2, 128), torch.bfloat16, rng, gpu), mixed((5, 2, 128), torch.bfloat16, rng, gpu)
    tables = i32([2, 5], gpu), i32([0, 2], gpu), i32([3], gpu)
    ai, a, b = i32([0, 5], gpu), i32([1, 4], gpu), i32([0, 3], gpu)

    def step(small, back):
        mx.append_paged_kv_cache_mx_indptr(k, v, ai, small[0], *tables)
        mx.quantize_pages(plain, a, small, b)
        mx.dequantize_pages(small, i32_52, back, a)

    i32_52 = i32([5, 2], gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(small, back)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(small, back)
    for seed in range(4):
        rng = np.random.default_rng(seed)
        k.copy_(mixed(k.shape, k.dtype, rng, gpu))
        plain[1].copy_(mixed(plain[1].shape, plain[1].dtype, rng, gpu))
        want_s, want_b = [t.clone() for t in small], [t.clone() for t in back]
        step(want_s, want_b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(small + back, want_s + want_b):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantised_pages_travel_with_their_scales(gpu, fmt):
    """move, a transfer buffer and a swap carry quantised pages as they are."""
    rng = np.random.default_rng(4)
    plain, small = pools(3, 8, 16, 2, 64, fmt, torch.float16, rng, gpu)
    mx.quantize_pages(plain, [1, 5, 2], small, [0, 3, 7])
    other = [torch.zeros_like(t) for t in small]
    ops.move(small, [0, 3, 7], other, [4, 1, 2])
    ops.unpack(ops.pack(small, [3]), other, [6])
    space = SwapSpace(ops.PagedPool(other), num_host_pages=4)
    space.swap_out("r", [4, 1])
    space.swap_in("r", [0, 5])
    torch.cuda.synchronize()
    a, b = [torch.zeros_like(t) for t in plain], [torch.zeros_like(t) for t in plain]
    mx.dequantize_pages(small, [0, 3, 7, 3], a, [0, 1, 2, 3])
    mx.dequantize_pages(other, [0, 5, 2, 6], b, [0, 1, 2, 3])
    for x, y in zip(a, b):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))
