"""Cases of the operators on a paged KV cache held in 16, 8 or 4 bits: its writers,
its conversions and the attention that reads it.

`kind` says which part of a serving program a case stands for:

  append      a step's new K/V rows go into a cache of 8-bit elements
              (append_paged_kv_cache_mx and its fused form)
  quantize    the pages of requests go from a 16-bit pool to an 8-bit one, all
              layers in one call (quantize_pages): a prefill instance hands
              requests over to a decode instance with a smaller cache
  dequantize  and back (dequantize_pages)
  park        both, through 4 bits: a preempted request kept small, then resumed
  attend      attention of each request's last tokens over its pages
              (paged_attention): single tokens, or a tree of drafted ones
  step        a layer of a verification step: append to a quantised cache, then
              attend over it

The quantised format: blocks of 32 elements along head_dim share the smallest
power of two that brings the block's largest magnitude within the element type
(e4m3 up to 448, e2m1 up to 6), between 2^-117 and 2^127; elements are rounded
to nearest even; a block with a non-finite value has the scale byte 255 and
reads as NaN.  Half a page (its keys or its values) is [page, heads, head_dim]
elements (4-bit ones two to a byte, the even one low), then [page, heads,
head_dim / 32] scale bytes (exponent + 127).

Attention: a request's last tokens are its queries.  Each sees every earlier
token, and those of the last tokens that its row of the tree mask has a bit for
(bit j % 64 of word j // 64; without a mask: itself and those before it).
"""
import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
ELEM = {"float16": 2, "bfloat16": 2, "float32": 4, "mxfp8": 33 / 32, "mxfp4": 17 / 32}
BLOCK = 32
TOP = {"mxfp8": 448.0, "mxfp4": 6.0}
LLAMA3 = dict(heads=8, head_dim=128, page=16, dtype="bfloat16")
LLAMA3_TP8 = dict(LLAMA3, heads=1)
LLAMA2_7B = dict(LLAMA3, heads=32, dtype="float16")


def listed():
    return [
        # A decode step of 64 running requests: one token each, where latency is all.
        dict(LLAMA3, name="append_decode_64req", kind="append", requests=64, tokens=1, ragged=False, context=1000,
             fused=True, strided=False),
        # A prefill batch; K and V are slices of the fused QKV projection.
        dict(LLAMA3, name="append_prefill_16x1024", kind="append", requests=16, tokens=1024, ragged=True, context=0,
             fused=True, strided=True),
        # Multi-head attention without grouped KV heads; chunked prefill at
        # unaligned positions, positions computed once per step.
        dict(LLAMA2_7B, name="append_prefill_2x4095_7b", kind="append", requests=2, tokens=4095, ragged=False,
             context=777, fused=False, strided=False),
        # One 512-token request handed over.
        dict(LLAMA3, name="quantize_512tok", kind="quantize", layers=32, requests=1, tokens=512, format="mxfp8"),
        # A batch handed over on one GPU of a tensor-parallel group: 8 KiB pages.
        dict(LLAMA3_TP8, name="quantize_16req_tp8", kind="quantize", layers=80, requests=16, tokens=2048,
             format="mxfp8"),
        # One long request read back.
        dict(LLAMA3, name="dequantize_4096tok", kind="dequantize", layers=32, requests=1, tokens=4096,
             format="mxfp8"),
        # A preempted request through 4 bits and back.
        dict(LLAMA2_7B, name="park_1000tok_7b", kind="park", layers=32, requests=1, tokens=1000, format="mxfp4"),
        # One user's next token early in an answer: the smallest call.
        dict(LLAMA3, name="decode_1x512", kind="attend", requests=1, context=512, tokens=1, ragged=False, tree=False,
             group=4, cache="bfloat16", cap=0.0),
        # A full decode batch of ragged requests.
        dict(LLAMA3, name="decode_256req", kind="attend", requests=256, context=2048, tokens=1, ragged=True,
             tree=False, group=8, cache="bfloat16", cap=0.0),
        # Large trees of drafted tokens over an 8-bit cache: the most work per byte.
        dict(LLAMA3, name="tree_8x4096_mxfp8", kind="attend", requests=8, context=4096, tokens=63, ragged=False,
             tree=True, group=8, cache="mxfp8", cap=0.0),
        # A small tree over one long context, no grouped heads: split over its length.
        dict(LLAMA2_7B, name="tree_1x32768_7b", kind="attend", requests=1, context=32768, tokens=12, ragged=False,
             tree=True, group=1, cache="float16", cap=0.0),
        # A verification step of ragged drafts over a 4-bit cache, with capped scores.
        dict(LLAMA3, name="step_16req_mxfp4", kind="step", requests=16, context=8000, tokens=9, ragged=True,
             tree=True, group=4, cache="mxfp4", cap=30.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        kind = rng.choice(["append", "append", "quantize", "dequantize", "park", "attend", "attend", "attend", "step"])
        case = dict(kind=kind, heads=rng.choice([1, 2, 3, 5, 8, 16, 32]), head_dim=rng.choice([64, 128, 128, 256]),
                    page=rng.choice([16, 16, 16, 32, 24, 64]), dtype=rng.choice(["bfloat16", "float16"]))
        if kind == "append":
            case.update(requests=_log_int(rng, 1, 256), tokens=_log_int(rng, 1, 8192), ragged=rng.random() < 0.5,
                        context=rng.choice([0, rng.randint(1, 4000)]), fused=rng.random() < 0.6,
                        strided=rng.random() < 0.4, dtype=rng.choice(["bfloat16", "float16", "float32"]))
        elif kind in ("quantize", "dequantize", "park"):
            case.update(layers=_log_int(rng, 1, 80), requests=_log_int(rng, 1, 64), tokens=_log_int(rng, 1, 8192),
                        format="mxfp4" if kind == "park" else "mxfp8",
                        dtype=rng.choice(["bfloat16", "float16", "float32"]))
        else:
            case.update(requests=_log_int(rng, 1, 256), context=_log_int(rng, 1, 65536),
                        tokens=rng.choice([1, _log_int(rng, 1, 256)]), ragged=rng.random() < 0.5,
                        tree=rng.random() < 0.6, group=rng.choice([1, 2, 3, 4, 7, 8, 16]),
                        cap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                        cache=rng.choice(["mxfp8", "mxfp4"] + ([case["dtype"]] * 2 if kind == "attend" else [])))
            # room for the scores of the plain form
            if case["requests"] * case["heads"] * case["group"] * case["tokens"] * case["context"] > 2e9:
                continue
            if case["requests"] * case["heads"] * case["head_dim"] * (case["context"] + case["tokens"]) > 1.2e9:
                continue
        w = work(case)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return case


def _lengths(case):
    """(tokens before this call, tokens of this call) of each request."""
    rng = np.random.default_rng(case["requests"] * 1009 + case.get("context", 0) * 31 + case["tokens"])
    n = case["requests"]
    ctx = np.full(n, case.get("context", 0), np.int64)
    new = np.full(n, case["tokens"], np.int64)
    if case.get("ragged"):
        ctx = rng.integers(ctx // 32, ctx + 1)
        new = rng.integers((new + 3) // 4, new + 1)
    return ctx, new


def work(case):
    H, D = case["heads"], case["head_dim"]
    ctx, new = _lengths(case)
    if case["kind"] == "append":
        n = int(new.sum()) * H * D * 2
        return {"bytes": n * (ELEM[case["dtype"]] + ELEM["mxfp8"]), "flops": 0}
    if case["kind"] in ("quantize", "dequantize", "park"):
        pages = int((-(-new // case["page"])).sum())
        n = case["layers"] * pages * 2 * case["page"] * H * D
        return {"bytes": n * (ELEM[case["dtype"]] + ELEM[case["format"]]) * (2 if case["kind"] == "park" else 1),
                "flops": 0}
    rows = int(new.sum()) * H * case["group"]
    seen = int(((ctx + new) * new).sum()) * H * case["group"]
    n = int((ctx + new).sum()) * H * 2 * D * ELEM[case["cache"]]
    n += rows * (2 * D * ELEM[case["dtype"]] + 4)
    if case["kind"] == "step":
        n += int(new.sum()) * H * D * 2 * (ELEM[case["dtype"]] + ELEM[case["cache"]])
    return {"bytes": n, "flops": 4 * seen * D}


# ---------------------------------------------------------------- plain forms

def _quantize(x, fmt):
    """(elements, scale bytes) of x [..., D] float32: e4m3 as bytes, e2m1 packed."""
    b = x.unflatten(-1, (-1, BLOCK))
    amax = b.abs().amax(-1)
    bits = amax.view(torch.int32)
    # exponent of the smallest power of two that leaves amax / 2^e <= TOP
    lead, mant = (8, 0x600000) if fmt == "mxfp8" else (2, 0x400000)
    byte = (((bits >> 23) - lead + ((bits & 0x7FFFFF) > mant)).clamp(10, 254)).to(torch.int32)
    byte = torch.where(torch.isfinite(b).all(-1), byte, 255)
    inv = torch.ldexp(torch.ones_like(amax), 127 - byte)
    y = torch.where((byte == 255).unsqueeze(-1), torch.zeros_like(b), b * inv.unsqueeze(-1))
    byte = byte.to(torch.uint8)
    if fmt == "mxfp8":
        return y.flatten(-2).to(torch.float8_e4m3fn).view(torch.uint8), byte
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5))
    code = (code + 8 * torch.signbit(y)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte


def _values(data, byte, fmt):
    """float32 values [..., D] of elements [..., D or D / 2] and scale bytes [..., D / 32]."""
    if fmt == "mxfp8":
        e = data.view(torch.float8_e4m3fn).float()
    else:
        code = torch.stack([data & 15, data >> 4], -1).flatten(-2).int()
        mag, ex = code & 1, (code >> 1) & 3
        e = torch.where(ex > 0, torch.ldexp(1 + 0.5 * mag.float(), ex - 1), 0.5 * mag.float())
        e = torch.where(code >= 8, -e, e)
    scale = torch.ldexp(torch.ones(byte.shape, device=byte.device), byte.int() - 127)
    scale = torch.where(byte == 255, math.nan, scale)
    return (e.unflatten(-1, (-1, BLOCK)) * scale.unsqueeze(-1)).flatten(-2)


def _row(D, fmt):
    return (D if fmt == "mxfp8" else D // 2) + D // BLOCK


def _halves(cache, D, fmt):
    """Views of quantised caches [..., P, H, R]: elements [..., P, H, D or D / 2] and
    scale bytes [..., P, H, D / 32]."""
    P, H, R = cache.shape[-3:]
    flat = cache.flatten(-3)
    per = R - D // BLOCK
    return (flat[..., :P * H * per].unflatten(-1, (P, H, per)),
            flat[..., P * H * per:].unflatten(-1, (P, H, D // BLOCK)))


def _typed(cache, D):
    """A cache of 8-bit elements as the values that its bytes stand for."""
    data, byte = _halves(cache, D, "mxfp8")
    return {"elements": data.view(torch.float8_e4m3fn), "scales": byte.view(torch.float8_e8m0fnu)}


def _slots(s):
    """Page and slot of each new token."""
    at = torch.arange(s.nnz, device=s.dev)
    b = torch.searchsorted(s.qo_indptr[1:].long(), at, right=True)
    pages = (s.kv_indptr[1:] - s.kv_indptr[:-1])[b]
    length = (pages - 1).clamp(min=0) * s.P + s.last[b]
    pos = length - (s.qo_indptr[b + 1] - s.qo_indptr[b]) + (at - s.qo_indptr[b])
    return s.kv_indices[(s.kv_indptr[b] + pos // s.P).long()].long(), (pos % s.P).long()


def _append(s):
    data, byte = _halves(s.cache, s.D, s.fmt)
    page, slot = _slots(s)
    e, c = _quantize(torch.stack([s.key, s.value], 1).float(), s.fmt)
    data[page, :, slot] = e
    byte[page, :, slot] = c


def _attend(s):
    D, H, G, B, P = s.D, s.heads, s.group, s.requests, s.P
    n_new = s.qo_indptr[1:] - s.qo_indptr[:-1]
    length = ((s.kv_indptr[1:] - s.kv_indptr[:-1] - 1).clamp(min=0) * P + s.last).long()
    base = length - n_new
    p = torch.arange(s.max_len, device=s.dev)
    at = (s.kv_indptr[:-1, None] + p[None, :] // P).clamp(max=s.kv_indices.numel() - 1)
    page, slot = s.kv_indices[at.long()].long(), (p % P)[None, :].expand(B, -1)
    if s.fmt is None:
        kv = s.cache[page, :, slot].float()
    else:
        data, byte = _halves(s.cache, D, s.fmt)
        kv = _values(data[page, :, slot], byte[page, :, slot], s.fmt)
    kv = kv.permute(2, 0, 3, 1, 4)                                        # [2, B, H, M, D]
    j = torch.arange(s.max_new, device=s.dev)
    row = (s.qo_indptr[:-1, None] + j[None, :]).clamp(max=s.nnz - 1).long()
    q = s.q[row].float().unflatten(2, (H, G)).permute(0, 2, 1, 3, 4).reshape(B, H, s.max_new * G, D)
    x = torch.matmul(q, kv[0].transpose(-1, -2).contiguous()) * s.scale   # [B, H, T * G, M]
    if s.cap > 0:
        x = s.cap * torch.tanh(x / s.cap)
    d = p[None, :] - base[:, None]                                        # which of the new tokens, < 0: before them
    if s.mask is not None:
        words = s.mask[row]                                               # [B, T, W]
        w = torch.gather(words, 2, (d.clamp(0, 64 * words.shape[2] - 1) // 64)[:, None, :].expand(-1, s.max_new, -1))
        sees = ((w >> (d.clamp(min=0) % 64)[:, None, :]) & 1).bool()
    else:
        sees = d[:, None, :] <= j[None, :, None]
    sees = (sees & (d < n_new[:, None])[:, None, :]) | (d < 0)[:, None, :]
    sees = sees[:, None, :, None, :].expand(B, 1, s.max_new, G, s.max_len).reshape(B, 1, s.max_new * G, s.max_len)
    x = torch.where(sees, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x, kv[1].contiguous()) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total)).squeeze(-1)
    b = torch.searchsorted(s.qo_indptr[1:].long(), torch.arange(s.nnz, device=s.dev), right=True)
    t = torch.arange(s.nnz, device=s.dev) - s.qo_indptr[b]
    o = o.unflatten(2, (s.max_new, G)).permute(0, 2, 1, 3, 4)[b, t.long()]
    lse = lse.unflatten(2, (s.max_new, G)).permute(0, 2, 1, 3)[b, t.long()]
    return {"out": o.flatten(1, 2).to(s.dtype), "lse": lse.flatten(1, 2)}


def _to_quantised(s):
    for a, b in zip(s.plain, s.small):                                    # layer by layer
        data, byte = _halves(b, s.D, s.fmt)
        data[s.small_ids.long()], byte[s.small_ids.long()] = _quantize(a[s.plain_ids.long()].float(), s.fmt)


def _to_plain(s, out, ids):
    for a, b in zip(s.small, out):
        data, byte = _halves(a, s.D, s.fmt)
        b[ids.long()] = _values(data[s.small_ids.long()], byte[s.small_ids.long()], s.fmt).to(s.dtype)


# ---------------------------------------------------------------- inputs

def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _gen(seed, dev):
    return torch.Generator(device=dev).manual_seed(int(seed) * 2 + 1)


def _rows(shape, g, dev, dtype):
    """Keys or values as models have them: normal, a few channels many times larger."""
    x = torch.randn(shape, generator=g, device=dev, dtype=torch.float32)
    gain = torch.exp(0.5 * torch.randn(shape[-2:], generator=g, device=dev))
    return (x * gain).to(dtype)


def _stale_mx(cache, D, fmt, g):
    """Fills a quantised cache as one that has been in use: every byte an ordinary one."""
    cache.copy_(torch.randint(0, 256, cache.shape, generator=g, device=cache.device, dtype=torch.uint8))
    data, byte = _halves(cache, D, fmt)
    if fmt == "mxfp8":
        data.bitwise_and_(0xF7)                                            # no NaN
    byte.bitwise_and_(7).add_(116)


def _fill_mx(cache, D, fmt, g):
    data, byte = _halves(cache, D, fmt)
    N, _, P, H, _ = cache.shape
    step = max(1, (1 << 26) // (2 * P * H * D))
    for i in range(0, N, step):
        n = min(step, N - i)
        x = _rows((n, 2, P, H, D), g, cache.device, torch.float32)
        data[i:i + n], byte[i:i + n] = _quantize(x, fmt)


def _tree(new, words, rng):
    """Rows of bits: each drafted token sees itself and its ancestors; parents
    are drawn from the eight tokens before it."""
    B, T = len(new), int(new.max())
    rows = np.zeros((B, T, words), np.uint64)
    for i in range(T):
        if i:
            parent = i - 1 - rng.integers(0, min(i, 8), B)
            rows[:, i] = rows[np.arange(B), parent]
        rows[:, i, i // 64] |= np.uint64(1 << (i % 64))
    return np.concatenate([rows[b, :new[b]] for b in range(B)]).view(np.int64)


def prepare(case, seed):
    dev = _device()
    g, rng = _gen(seed, dev), np.random.default_rng(seed)
    dtype = DTYPES[case["dtype"]]
    H, D, P = case["heads"], case["head_dim"], case["page"]
    ctx, new = _lengths(case)
    s = SimpleNamespace(kind=case["kind"], dev=dev, dtype=dtype, heads=H, D=D, P=P, requests=case["requests"])

    def i32(x):
        return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)

    if s.kind in ("quantize", "dequantize", "park"):
        s.fmt = case["format"]
        n = int((-(-new // P)).sum())
        pool = n + 7
        s.small_ids, s.plain_ids, s.back_ids = (i32(rng.permutation(pool)[:n]) for _ in range(3))
        # pools as a program has them: one allocation, a view for each layer
        s.small_pool = torch.empty((case["layers"], pool, 2, P, H, _row(D, s.fmt)), device=dev, dtype=torch.uint8)
        s.small = list(s.small_pool)
        for c in s.small:
            (_fill_mx if s.kind == "dequantize" else _stale_mx)(c, D, s.fmt, g)
        if s.kind != "dequantize":
            s.plain = [_rows((pool, 2, P, H, D), g, dev, dtype) for _ in range(case["layers"])]
        if s.kind != "quantize":
            s.back_pool = torch.zeros((case["layers"], pool, 2, P, H, D), device=dev, dtype=dtype)
            s.back = list(s.back_pool)
        return s

    total = ctx + new
    pages = -(-total // P)
    pool = int(pages.sum()) + 7
    s.nnz = int(new.sum())
    s.kv_indices = i32(rng.permutation(pool)[:int(pages.sum())])
    s.kv_indptr = i32(np.concatenate([[0], np.cumsum(pages)]))
    s.last = i32((total - 1) % P + 1)
    s.qo_indptr = i32(np.concatenate([[0], np.cumsum(new)]))
    s.max_len, s.max_new = int(total.max()), int(new.max())
    if s.kind in ("append", "step"):
        if case.get("strided"):
            qkv = _rows((s.nnz, 6 * H, D), g, dev, dtype)
            s.key, s.value = qkv[:, 4 * H:5 * H], qkv[:, 5 * H:]
        else:
            s.key, s.value = _rows((s.nnz, H, D), g, dev, dtype), _rows((s.nnz, H, D), g, dev, dtype)
    if s.kind == "append":
        s.fmt, s.fused = "mxfp8", case["fused"]
        s.cache = torch.empty((pool, 2, P, H, _row(D, s.fmt)), device=dev, dtype=torch.uint8)
        _stale_mx(s.cache, D, s.fmt, g)
        return s
    s.group, s.cap, s.scale = case["group"], case["cap"], 1 / math.sqrt(D)
    s.fmt = case["cache"] if case["cache"].startswith("mx") else None
    # scores that spread over a few units, as trained heads' do
    s.q = (1.5 * torch.randn((s.nnz, H * s.group, D), generator=g, device=dev)).to(dtype)
    if s.fmt:
        s.cache = torch.empty((pool, 2, P, H, _row(D, s.fmt)), device=dev, dtype=torch.uint8)
        _fill_mx(s.cache, D, s.fmt, g)
    else:
        s.cache = _rows((pool, 2, P, H, D), g, dev, dtype)
    words = -(-s.max_new // 64)
    s.mask = torch.from_numpy(_tree(new, words, rng)).to(dev) if case["tree"] else None
    return s


def run(s):
    if own:
        from paceserve_amd.kv_transfer import attention, mx
        from paceserve_amd.kv_transfer import append as ap
        if s.kind == "quantize":
            mx.quantize_pages(s.plain, s.plain_ids, s.small, s.small_ids)
            return _typed(s.small_pool, s.D)
        if s.kind == "dequantize":
            mx.dequantize_pages(s.small, s.small_ids, s.back, s.back_ids)
            return s.back_pool
        if s.kind == "park":
            mx.quantize_pages(s.plain, s.plain_ids, s.small, s.small_ids)
            mx.dequantize_pages(s.small, s.small_ids, s.back, s.back_ids)
            return s.back_pool
        if s.kind == "append" and not s.fused:
            seq = ap.get_seq_lens(s.kv_indptr, s.last, s.P)
            bi, pos = ap.get_batch_indices_positions(s.qo_indptr, seq, s.nnz)
            mx.append_paged_kv_cache_mx(s.key, s.value, bi, pos, s.cache, s.kv_indices, s.kv_indptr, s.last)
            return _typed(s.cache, s.D)
        if s.kind in ("append", "step"):
            mx.append_paged_kv_cache_mx_indptr(s.key, s.value, s.qo_indptr, s.cache, s.kv_indices, s.kv_indptr,
                                               s.last)
            if s.kind == "append":
                return _typed(s.cache, s.D)
        out, lse = attention.paged_attention(s.q, s.cache, s.kv_indices, s.kv_indptr, s.last, s.qo_indptr,
                                             max_q_len=s.max_new, tree_mask=s.mask, sm_scale=s.scale,
                                             logits_soft_cap=s.cap, return_lse=True)
        return {"out": out, "lse": lse}
    if s.kind == "quantize":
        _to_quantised(s)
        return _typed(s.small_pool, s.D)
    if s.kind == "dequantize":
        _to_plain(s, s.back, s.back_ids)
        return s.back_pool
    if s.kind == "park":
        _to_quantised(s)
        _to_plain(s, s.back, s.back_ids)
        return s.back_pool
    if s.kind in ("append", "step"):
        _append(s)
        if s.kind == "append":
            return _typed(s.cache, s.D)
    return _attend(s)


# ---------------------------------------------------------------- 64 bits

def _block_scale64(x, fmt):
    """Exponents [..., D / 32] of float64 rows, or None-like 1000 for a block that reads as NaN."""
    b = x.unflatten(-1, (-1, BLOCK))
    m, e = torch.frexp(b.abs().amax(-1) / TOP[fmt])                       # m in [0.5, 1)
    e = torch.where(m > 0.5, e, e - 1).double()
    e = torch.where(m == 0, -117.0, e).clamp(-117, 127)
    return torch.where(torch.isfinite(b).all(-1), e, 1000.0)


def _round64(x, e, fmt):
    """Elements that x [..., D] rounds to under block exponents e, as float64."""
    y = x.unflatten(-1, (-1, BLOCK)) * torch.exp2(-e).unsqueeze(-1)
    low, bits = (-6, 3) if fmt == "mxfp8" else (0, 1)
    ex = torch.frexp(y.abs())[1].double() - 1
    step = torch.exp2(torch.where(y == 0, float(low), ex).clamp(min=low) - bits)
    return torch.where((e < 1000).unsqueeze(-1), torch.round(y / step) * step, 0.0)


def _read64(cache, D, fmt):
    """float64 values of a quantised cache, byte by byte from the definition."""
    N, _, P, H, R = cache.shape
    flat = cache.reshape(N, 2, -1)
    cut = P * H * (R - D // BLOCK)
    codes = torch.arange(256, dtype=torch.int64)
    if fmt == "mxfp8":
        ex, man = (codes >> 3) & 15, (codes & 7).double()
        table = torch.where(ex > 0, (1 + man / 8) * torch.exp2(ex.double() - 7), man / 8 * 2.0 ** -6)
        table = torch.where(codes > 127, -table, table)
        e = table.to(cache.device)[flat[:, :, :cut].long()]
    else:
        table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
        table = torch.cat([table, -table]).to(cache.device)
        b = flat[:, :, :cut].long()
        e = torch.stack([table[b % 16], table[b // 16]], -1).flatten(-2)
    c = flat[:, :, cut:].double() - 127
    scale = torch.where(c == 128, math.nan, torch.exp2(c))
    return (e.unflatten(-1, (-1, BLOCK)) * scale.unsqueeze(-1)).reshape(N, 2, P, H, D)


def _written64(old, page, slot, x):
    """The typed outputs of a cache of 8-bit elements whose rows (page, slot) became x (float64)."""
    N, _, P, H, R = old.shape
    D = x.shape[-1]
    flat = old.reshape(N, 2, -1)
    el = flat[:, :, :P * H * D].view(torch.float8_e4m3fn).double().reshape(N, 2, P, H, D)
    sc = torch.exp2(flat[:, :, P * H * D:].double() - 127).reshape(N, 2, P, H, D // BLOCK)
    e = _block_scale64(x, "mxfp8")
    v = _round64(x, e, "mxfp8").flatten(-2)
    e = torch.where(e < 1000, torch.exp2(e), math.nan)
    if slot is None:
        el[page], sc[page] = v, e
    else:
        el[page, :, slot], sc[page, :, slot] = v, e
    return {"elements": el, "scales": sc}


def _attend64(s, cache):
    """Each request and head by itself, in float64."""
    ip, ix, qo = s.kv_indptr.tolist(), s.kv_indices.long(), s.qo_indptr.tolist()
    out = torch.zeros((s.nnz, s.heads * s.group, s.D), dtype=torch.float64, device=s.dev)
    lse = torch.zeros((s.nnz, s.heads * s.group), dtype=torch.float64, device=s.dev)
    for b, last in enumerate(s.last.tolist()):
        kv = cache[ix[ip[b]:ip[b + 1]]]
        kv = (kv.double() if s.fmt is None else _read64(kv, s.D, s.fmt)).transpose(0, 1).flatten(1, 2)
        n, t = (ip[b + 1] - ip[b] - 1) * s.P + last, qo[b + 1] - qo[b]
        hidden = torch.zeros((t, n), dtype=torch.bool, device=s.dev)
        tail = torch.ones((t, t), dtype=torch.bool, device=s.dev).triu(1)
        if s.mask is not None:
            bit = torch.arange(64, device=s.dev)
            tail = ((s.mask[qo[b]:qo[b + 1], :, None] >> bit) & 1).flatten(1)[:, :t] == 0
        hidden[:, n - t:] = tail
        for h in range(s.heads):
            hs = slice(h * s.group, (h + 1) * s.group)
            x = s.q[qo[b]:qo[b + 1], hs].double().flatten(0, 1) @ kv[0, :n, h].T * s.scale
            if s.cap > 0:
                x = s.cap * torch.tanh(x / s.cap)
            x = x.masked_fill(hidden.repeat_interleave(s.group, 0), -math.inf)
            out[qo[b]:qo[b + 1], hs] = (torch.softmax(x, -1) @ kv[1, :n, h]).unflatten(0, (t, s.group))
            lse[qo[b]:qo[b + 1], hs] = torch.logsumexp(x, -1).unflatten(0, (t, s.group))
    return {"out": out, "lse": lse}


def exact(case, seed):
    w = work(case)
    if w["flops"] > 1e12 or case["requests"] * case["heads"] > 4200 and case["kind"] in ("attend", "step"):
        return None
    s = prepare(case, seed)
    if s.kind == "quantize":
        got = [_written64(b, s.small_ids.long(), None, a[s.plain_ids.long()].double())
               for a, b in zip(s.plain, s.small)]
        return {k: torch.stack([x[k] for x in got]) for k in got[0]}
    if s.kind in ("dequantize", "park"):
        out = []
        for i in range(len(s.back)):
            if s.kind == "park":
                x = s.plain[i][s.plain_ids.long()].double()
                e = _block_scale64(x, s.fmt)
                v = (_round64(x, e, s.fmt) * torch.exp2(e).unsqueeze(-1)).flatten(-2)
            else:
                v = _read64(s.small[i][s.small_ids.long()], s.D, s.fmt)
            o = s.back[i].double()
            o[s.back_ids.long()] = v
            out.append(o)
        return torch.stack(out)
    if s.kind in ("append", "step"):
        at = [(s.kv_indptr[b].item(), int(n), s.qo_indptr[b].item(), s.qo_indptr[b + 1].item())
              for b, n in enumerate(((s.kv_indptr[1:] - s.kv_indptr[:-1] - 1) * s.P + s.last).tolist())]
        pos = [(first, n - (a1 - a0) + i) for first, n, a0, a1 in at for i in range(a1 - a0)]
        first, p = torch.tensor(pos, device=s.dev).T
        page, slot = s.kv_indices.long()[first + p // s.P], p % s.P
        x = torch.stack([s.key, s.value], 1).double()
        if s.kind == "append":
            return _written64(s.cache, page, slot, x)
        e = _block_scale64(x, s.fmt)
        v = _round64(x, e, s.fmt).flatten(-2)
        data, byte = _halves(s.cache, s.D, s.fmt)
        byte[page, :, slot] = (e + 127).to(torch.uint8)
        if s.fmt == "mxfp8":
            data[page, :, slot] = v.to(torch.float8_e4m3fn).view(torch.uint8)  # exact: v is such a value
        else:
            grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=s.dev)
            code = torch.searchsorted(grid, v.abs()) + 8 * torch.signbit(v)
            data[page, :, slot] = (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8)
    return _attend64(s, s.cache)
