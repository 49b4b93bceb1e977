"""Cases of the operators around a paged cache that a layer of a serving step
runs beside the append and the attention: the tables of a batch, queries and
keys normalised and rotated on their way into the pages, and attention over a
cache of latent vectors.

`kind` says which operator a case stands for:

  tables   page lists, positions and slots of a batch from its lengths
           (build_tables)
  rotate   each head's queries and keys normalised, then rotated by position
           (norm_rotate)
  write    the same on the way into the cache, with the values
           (append_paged_kv_cache_rope): a 16-bit cache or a quantised one
  latent   a token's latent vector normalised and its shared key part rotated,
           into a latent cache (append_paged_latent_cache)
  absorbed attention of each request's last tokens over a latent cache
           (paged_latent_attention): keys are the rows [latent, rotated part],
           values their latent part, the same ones for every head
  prompt   attention of prompts over keys and values expanded from the latents,
           with the rotated part of the keys shared by the heads
           (latent_prompt_attention)

A row x of a head is normalised as x / sqrt(mean(x^2) + eps) * weight.  The
rotation takes the pair (a, b) at (i, i + r / 2), or (2 i, 2 i + 1) if
interleaved, to (a cos - b sin, b cos + a sin); r columns of the row rotate, and
a table [positions, r] holds the r / 2 cosines of a position, then its sines.  A
token with slot -1 is padding.  A latent cache is [pages, page, latent + 64].
"""
import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
ELEM = {"float16": 2, "bfloat16": 2, "mxfp8": 33 / 32}
BLOCK, ROPE, EPS = 32, 64, 1e-6
LLAMA3 = dict(q_heads=32, heads=8, head_dim=128, rotary=128, page=16, dtype="bfloat16")
LATENT = dict(latent=512, page=16, dtype="bfloat16")


def listed():
    return [
        # A decode step of 64 running requests: launch and latency.
        dict(name="tables_decode_64req", kind="tables", requests=64, context=1000, tokens=1, ragged=True, page=16),
        # A ragged prefill step of many requests with long page lists.
        dict(name="tables_prefill_512req", kind="tables", requests=512, context=8192, tokens=100, ragged=True, page=16),
        # A prefill batch whose heads are normalised; q and k are slices of one projection.
        dict(LLAMA3, name="rotate_prefill_16384tok", kind="rotate", tokens=16384, norm=True, strided=True,
             interleaved=False),
        # A decode step's rows into a 16-bit cache, without norms.
        dict(LLAMA3, name="write_decode_64tok", kind="write", tokens=64, norm=False, strided=True, interleaved=False,
             cache="bfloat16"),
        # A prefill batch into an 8-bit cache, with norms.
        dict(LLAMA3, name="write_prefill_8190tok_mxfp8", kind="write", tokens=8190, norm=True, strided=True,
             interleaved=False, cache="mxfp8"),
        # A decode step's latent rows.
        dict(LATENT, name="latent_decode_128tok", kind="latent", tokens=128, interleaved=True),
        # A prefill batch's.
        dict(LATENT, name="latent_prefill_16384tok", kind="latent", tokens=16384, interleaved=True),
        # One user's next token, on one GPU of a tensor-parallel group: the smallest call.
        dict(LATENT, name="absorbed_1x2000_16heads", kind="absorbed", requests=1, context=2000, tokens=1, heads=16,
             ragged=False, tree=False),
        # A full decode batch there: the cache's bytes.
        dict(LATENT, name="absorbed_128req_16heads", kind="absorbed", requests=128, context=8192, tokens=1, heads=16,
             ragged=True, tree=False),
        # All heads on one GPU, with drafted tokens under a tree mask: matrix products.
        dict(LATENT, name="absorbed_32x4096_128heads", kind="absorbed", requests=32, context=4096, tokens=3, heads=128,
             ragged=False, tree=True),
        # A prefill batch of ragged prompts.
        dict(kind="prompt", name="prompt_8x2000_16heads", requests=8, context=0, tokens=2000, heads=16, nope=128,
             ragged=True, dtype="bfloat16"),
        # One long prompt's second half, over the first half's keys.
        dict(kind="prompt", name="prompt_4096_of_8192_32heads", requests=1, context=4096, tokens=4096, heads=32,
             nope=128, ragged=False, dtype="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        kind = rng.choice(["tables", "rotate", "write", "write", "latent", "absorbed", "absorbed", "prompt", "prompt"])
        case = dict(kind=kind, dtype=rng.choice(["bfloat16", "bfloat16", "float16"]))
        if kind != "prompt":
            case["page"] = rng.choice([16, 16, 16, 32, 24, 64, 1])
        if kind == "tables":
            del case["dtype"]
            case.update(requests=_log_int(rng, 1, 2048), context=_log_int(rng, 1, 32768), tokens=_log_int(rng, 1, 512),
                        ragged=rng.random() < 0.8)
        elif kind in ("rotate", "write"):
            dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
            heads = rng.choice([1, 2, 3, 4, 8, 16])
            case.update(tokens=_log_int(rng, 1, 32768), heads=heads, q_heads=heads * rng.choice([1, 2, 4, 7, 8]),
                        head_dim=dim, rotary=rng.choice([dim, dim, dim // 2 // 16 * 16]), norm=rng.random() < 0.6,
                        strided=rng.random() < 0.5, interleaved=rng.random() < 0.3)
            if kind == "write":
                fits = dim % 64 == 0 and case["rotary"] % 64 == 0
                case["cache"] = rng.choice([case["dtype"], "mxfp8"]) if fits else case["dtype"]
        elif kind == "latent":
            case.update(tokens=_log_int(rng, 1, 65536), latent=rng.choice([256, 512, 512]),
                        interleaved=rng.random() < 0.5)
        elif kind == "absorbed":
            case.update(requests=_log_int(rng, 1, 256), context=_log_int(rng, 1, 65536), latent=rng.choice([256, 512, 512]),
                        tokens=rng.choice([1, 1, rng.randint(2, 16)]), heads=rng.choice([1, 3, 8, 16, 32, 64, 128]),
                        ragged=rng.random() < 0.6, tree=rng.random() < 0.4)
            # room for the scores and the widened rows of the plain form
            if case["requests"] * case["heads"] * case["tokens"] * case["context"] > 2e9:
                continue
            if case["requests"] * (case["context"] + case["tokens"]) * (case["latent"] + ROPE) > 2e9:
                continue
        else:
            case.update(requests=_log_int(rng, 1, 32), context=rng.choice([0, 0, rng.randint(1, 4096)]),
                        tokens=_log_int(rng, 1, 8192), heads=rng.choice([1, 3, 8, 16, 32]), nope=rng.choice([64, 128, 128]),
                        ragged=rng.random() < 0.6)
            if case["requests"] * case["heads"] * case["tokens"] * (case["context"] + case["tokens"]) > 3e9:
                continue
        w = work(case)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return case


def _lengths(case):
    """(tokens before this call, tokens of this call) of each request."""
    rng = np.random.default_rng(case["requests"] * 1009 + case["context"] * 31 + case["tokens"])
    n = case["requests"]
    ctx, new = np.full(n, case["context"], np.int64), np.full(n, case["tokens"], np.int64)
    if case["ragged"]:
        ctx = rng.integers(ctx // 16, ctx + 1)
        new = rng.integers((new + 3) // 4, new + 1)
    return ctx, new


def work(case):
    kind = case["kind"]
    if kind in ("tables", "absorbed", "prompt"):
        ctx, new = _lengths(case)
    if kind == "tables":
        pages = -(-(ctx + new) // case["page"])
        width = int(pages.max())
        return {"bytes": 4 * int(pages.sum()) + 4 * len(ctx) * (width + 4) + 12 * int(new.sum()), "flops": 0}
    if kind == "rotate":
        n = case["tokens"] * (case["q_heads"] + case["heads"]) * case["head_dim"]
        return {"bytes": 4 * n + case["tokens"] * (4 * case["rotary"] + 4), "flops": 0}
    if kind == "write":
        n, kv = (case["tokens"] * h * case["head_dim"] for h in (case["q_heads"], 2 * case["heads"]))
        return {"bytes": 4 * n + (2 + ELEM[case["cache"]]) * kv + case["tokens"] * (4 * case["rotary"] + 12), "flops": 0}
    if kind == "latent":
        return {"bytes": case["tokens"] * (4 * (case["latent"] + ROPE) + 4 * ROPE + 12), "flops": 0}
    rows = int(new.sum()) * case["heads"]
    if kind == "absorbed":
        seen = int(((ctx + new) * new).sum()) * case["heads"]
        return {"bytes": 2 * int((ctx + new).sum()) * (case["latent"] + ROPE) + rows * (4 * case["latent"] + 2 * ROPE + 4),
                "flops": 2 * seen * (2 * case["latent"] + ROPE)}
    seen = int((ctx * new + new * (new + 1) // 2).sum()) * case["heads"]
    keys, nope = int((ctx + new).sum()), case["nope"]
    return {"bytes": rows * (4 * nope + 2 * ROPE + 4) + 2 * keys * (2 * nope * case["heads"] + ROPE),
            "flops": 2 * seen * (2 * nope + ROPE)}


# ---------------------------------------------------------------- plain forms

def _tables(s):
    pages = (s.seq_lens + s.P - 1) // s.P
    indptr = torch.cat([torch.zeros_like(pages[:1]), torch.cumsum(pages, 0)]).to(torch.int32)
    at = torch.arange(s.page_table.numel(), device=s.dev, dtype=torch.int32)
    b = torch.searchsorted(indptr[1:], at, right=True).clamp(max=s.requests - 1)
    i = (at - indptr[b]).clamp(max=s.page_table.shape[1] - 1).long()
    indices = torch.where(at < indptr[-1], s.page_table[b, i], -1)
    last = torch.where(s.seq_lens > 0, (s.seq_lens - 1) % s.P + 1, 0)
    token = torch.arange(s.nnz, device=s.dev, dtype=torch.int32)
    b = torch.searchsorted(s.qo_indptr[1:], token, right=True)
    pos = s.seq_lens[b] - s.qo_indptr[b + 1] + token
    slot = s.page_table[b, (pos // s.P).long()].long() * s.P + pos % s.P
    return {"kv_indices": indices, "kv_indptr": indptr, "kv_last_page_len": last.to(torch.int32),
            "positions": pos.to(torch.int32), "slot_mapping": slot}


def _norm(x, weight):
    x = x.float()
    if weight is None:
        return x
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()


def _rotate(x, positions, table, interleaved):
    """x [tokens, heads, D] float32; the table's columns rotate."""
    r = table.shape[1]
    cos, sin = table[positions.long()].unsqueeze(1).chunk(2, -1)
    head, tail = x[..., :r], x[..., r:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else head.chunk(2, -1)
    a, b = a * cos - b * sin, b * cos + a * sin
    head = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([head, tail], -1)


def _norm_rotate(s, x, weight):
    return _rotate(_norm(x, weight), s.positions, s.table, s.interleaved)


def _quantize(x):
    """(e4m3 bytes, scale bytes) of x [..., D] float32."""
    b = x.unflatten(-1, (-1, BLOCK))
    bits = b.abs().amax(-1).view(torch.int32)
    byte = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000)).clamp(10, 254)
    y = b * torch.ldexp(torch.ones_like(b[..., 0]), 127 - byte).unsqueeze(-1)
    return y.flatten(-2).to(torch.float8_e4m3fn).view(torch.uint8), byte.to(torch.uint8)


def _halves(cache, D):
    """Views of an 8-bit cache [..., P, H, R]: elements [..., P, H, D], scale bytes [..., P, H, D / 32]."""
    P, H, _ = cache.shape[-3:]
    flat = cache.flatten(-3)
    return flat[..., :P * H * D].unflatten(-1, (P, H, D)), flat[..., P * H * D:].unflatten(-1, (P, H, D // BLOCK))


def _typed(s):
    """A cache as the values that it holds."""
    if s.cache.dtype != torch.uint8:
        return s.cache
    data, byte = _halves(s.cache, s.D)
    return {"elements": data.view(torch.float8_e4m3fn), "scales": byte.view(torch.float8_e8m0fnu)}


def _write(s):
    q, k, v = _norm_rotate(s, s.q, s.q_weight), _norm_rotate(s, s.k, s.k_weight), s.v.float()
    page, slot = s.slot_mapping // s.P, s.slot_mapping % s.P
    kv = torch.stack([k, v], 1)
    if s.cache.dtype != torch.uint8:
        s.cache[page, :, slot] = kv.to(s.dtype)
    else:
        data, byte = _halves(s.cache, s.D)
        data[page, :, slot], byte[page, :, slot] = _quantize(kv)
    return {"q": q.to(s.dtype), "cache": _typed(s)}


def _latent(s):
    row = torch.cat([_norm(s.latent, s.weight),
                     _rotate(s.rope_key.float().unsqueeze(1), s.positions, s.table, s.interleaved).squeeze(1)], -1)
    s.cache[s.slot_mapping // s.P, s.slot_mapping % s.P] = row.to(s.dtype)
    return s.cache


def _softmax(x):
    """(weights, their sums, log-sum-exp) over the last dimension; rows that see nothing have sum 0."""
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    return x, total, (top + torch.log(total)).squeeze(-1)


def _absorbed(s):
    B, P = s.requests, s.P
    n_new = s.qo_indptr[1:] - s.qo_indptr[:-1]
    base = ((s.kv_indptr[1:] - s.kv_indptr[:-1] - 1) * P + s.last - n_new).long()
    p = torch.arange(s.max_len, device=s.dev)
    at = (s.kv_indptr[:-1, None] + p[None, :] // P).clamp(max=s.kv_indices.numel() - 1)
    kv = s.cache[s.kv_indices[at.long()].long(), (p % P)[None, :].expand(B, -1)].float()    # [B, M, L + 64]
    j = torch.arange(s.max_new, device=s.dev)
    row = (s.qo_indptr[:-1, None] + j[None, :]).clamp(max=s.nnz - 1).long()
    q = s.q[row].float().flatten(1, 2)                                                       # [B, T * H, L + 64]
    x = torch.matmul(q, kv.transpose(-1, -2).contiguous()) * s.scale
    d = p[None, :] - base[:, None]
    if s.mask is not None:
        bit = (s.mask[row][..., 0, None] >> d.clamp(0, 63)[:, None, :]) & 1
        sees = bit.bool()
    else:
        sees = d[:, None, :] <= j[None, :, None]
    sees = (sees & (d < n_new[:, None])[:, None, :]) | (d < 0)[:, None, :]
    x = torch.where(sees.repeat_interleave(s.heads, 1), x, -math.inf)
    x, total, lse = _softmax(x)
    o = torch.matmul(x, kv[..., :s.L].contiguous()) / torch.where(total > 0, total, 1.0)
    b = torch.searchsorted(s.qo_indptr[1:], torch.arange(s.nnz, device=s.dev, dtype=torch.int32), right=True)
    t = (torch.arange(s.nnz, device=s.dev) - s.qo_indptr[b]).long()
    return {"out": o.unflatten(1, (s.max_new, s.heads))[b, t].to(s.dtype),
            "lse": lse.unflatten(1, (s.max_new, s.heads))[b, t]}


def _padded(indptr, most, last):
    """Rows [B, most] of ragged sequences, those past a sequence's end held at `last`."""
    return (indptr[:-1, None] + torch.arange(most, device=indptr.device)[None, :]).clamp(max=last).long()


def _prompt(s):
    q_len, k_len = s.qo_indptr[1:] - s.qo_indptr[:-1], s.kv_indptr[1:] - s.kv_indptr[:-1]
    qrow, krow = _padded(s.qo_indptr, s.max_new, s.nnz - 1), _padded(s.kv_indptr, s.max_len, s.key.shape[0] - 1)
    q = s.q[qrow].float().permute(0, 2, 1, 3).contiguous()                                   # [B, H, T, D]
    k = torch.cat([s.key, s.rope_key.unsqueeze(1).expand(-1, s.heads, -1)], -1)[krow].float()
    x = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * s.scale                        # [B, H, T, M]
    i, p = torch.arange(s.max_new, device=s.dev), torch.arange(s.max_len, device=s.dev)
    sees = p[None, None, :] <= (k_len - q_len)[:, None, None] + i[None, :, None]
    x = torch.where(sees.unsqueeze(1), x, -math.inf)
    x, total, lse = _softmax(x)
    o = torch.matmul(x, s.value[krow].float().permute(0, 2, 1, 3).contiguous())
    o = o / torch.where(total > 0, total, 1.0)
    b = torch.searchsorted(s.qo_indptr[1:], torch.arange(s.nnz, device=s.dev, dtype=torch.int32), right=True)
    t = (torch.arange(s.nnz, device=s.dev) - s.qo_indptr[b]).long()
    return {"out": o[b, :, t].to(s.dtype), "lse": lse[b, :, t]}


# ---------------------------------------------------------------- inputs

def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _rows(shape, g, dev, dtype):
    """Projected rows as models have them: normal, a few channels many times larger."""
    x = torch.randn(shape, generator=g, device=dev)
    return (x * torch.exp(0.5 * torch.randn(shape[-1:], generator=g, device=dev))).to(dtype)


def _weight(n, g, dev, dtype):
    return (1 + 0.2 * torch.randn(n, generator=g, device=dev)).to(dtype)


def _rotary_table(positions, rotary, dev):
    angle = torch.arange(positions, device=dev, dtype=torch.float64)[:, None] * \
        10000.0 ** (-torch.arange(0, rotary, 2, device=dev, dtype=torch.float64) / rotary)
    return torch.cat([torch.cos(angle), torch.sin(angle)], -1).float()


def _tree(new, rng):
    """Rows of bits: each drafted token sees itself and its ancestors."""
    B, T = len(new), int(new.max())
    rows = np.zeros((B, T, 1), np.uint64)
    for i in range(T):
        if i:
            rows[:, i] = rows[np.arange(B), i - 1 - rng.integers(0, min(i, 4), B)]
        rows[:, i, 0] |= np.uint64(1 << i)
    return np.concatenate([rows[b, :new[b]] for b in range(B)]).view(np.int64)


def prepare(case, seed):
    dev = _device()
    g, rng = torch.Generator(device=dev).manual_seed(int(seed) * 2 + 1), np.random.default_rng(seed)
    kind = case["kind"]
    s = SimpleNamespace(kind=kind, dev=dev, P=case.get("page"))

    def i32(x):
        return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)

    if kind == "tables":
        ctx, new = _lengths(case)
        pages = -(-(ctx + new) // s.P)
        table = np.zeros((len(ctx), int(pages.max())), np.int64)
        at = np.concatenate([[0], np.cumsum(pages)])
        ids = rng.permutation(int(at[-1]) + 7)
        for b in range(len(ctx)):
            table[b, :pages[b]] = ids[at[b]:at[b + 1]]
        s.requests, s.nnz = len(ctx), int(new.sum())
        s.page_table, s.seq_lens = i32(table), i32(ctx + new)
        s.qo_indptr = i32(np.concatenate([[0], np.cumsum(new)]))
        return s
    s.dtype = DTYPES[case["dtype"]]
    if kind in ("rotate", "write", "latent"):
        n, s.interleaved = case["tokens"], case["interleaved"]
        far = 131072
        s.positions = i32(rng.integers(0, far, n))
        s.table = _rotary_table(far, case.get("rotary", ROPE), dev)
        if kind != "rotate":
            pool = -(-n // s.P) + 7
            s.slot_mapping = torch.tensor(rng.permutation(pool * s.P)[:n], dtype=torch.int64, device=dev)
    if kind == "latent":
        s.L = case["latent"]
        # both parts come out of one projection
        x = _rows((n, s.L + ROPE), g, dev, s.dtype)
        s.latent, s.rope_key = x[:, :s.L], x[:, s.L:]
        s.weight = _weight(s.L, g, dev, s.dtype)
        s.cache = _rows((pool, s.P, s.L + ROPE), g, dev, s.dtype)
        return s
    if kind in ("rotate", "write"):
        H, Hq, D = case["heads"], case["q_heads"], case["head_dim"]
        s.H, s.D = H, D
        if case["strided"]:
            s.q, s.k, s.v = _rows((n, Hq + 2 * H, D), g, dev, s.dtype).split([Hq, H, H], 1)
        else:
            s.q, s.k, s.v = (_rows((n, h, D), g, dev, s.dtype) for h in (Hq, H, H))
        s.q_weight, s.k_weight = (_weight(D, g, dev, s.dtype) if case["norm"] else None for _ in range(2))
        if kind == "write":
            if case["cache"] == "mxfp8":
                # a cache that has been in use: every byte an ordinary one
                s.cache = torch.randint(0, 256, (pool, 2, s.P, H, D + D // BLOCK), generator=g, device=dev,
                                        dtype=torch.uint8)
                data, byte = _halves(s.cache, D)
                data.bitwise_and_(0xF7)
                byte.bitwise_and_(7).add_(116)
            else:
                s.cache = _rows((pool, 2, s.P, H, D), g, dev, s.dtype)
        return s
    ctx, new = _lengths(case)
    s.requests, s.heads, s.nnz = len(ctx), case["heads"], int(new.sum())
    s.qo_indptr = i32(np.concatenate([[0], np.cumsum(new)]))
    s.max_len, s.max_new = int((ctx + new).max()), int(new.max())
    if kind == "absorbed":
        s.L = case["latent"]
        total = ctx + new
        pages = -(-total // s.P)
        pool = int(pages.sum()) + 7
        s.kv_indices = i32(rng.permutation(pool)[:int(pages.sum())])
        s.kv_indptr = i32(np.concatenate([[0], np.cumsum(pages)]))
        s.last = i32((total - 1) % s.P + 1)
        # latents are normalised, and absorbed queries give scores that spread over a few units
        s.cache = torch.randn((pool, s.P, s.L + ROPE), generator=g, device=dev).to(s.dtype)
        s.q = (1.5 * torch.randn((s.nnz, s.heads, s.L + ROPE), generator=g, device=dev)).to(s.dtype)
        s.scale = 1 / math.sqrt(s.L + ROPE)
        s.mask = torch.from_numpy(_tree(new, rng)).to(dev) if case["tree"] else None
        return s
    s.nope = case["nope"]
    s.kv_indptr = i32(np.concatenate([[0], np.cumsum(ctx + new)]))
    n = int((ctx + new).sum())
    # keys and values are the halves of one projection of the latents
    kv = torch.randn((n, s.heads, 2 * s.nope), generator=g, device=dev).to(s.dtype)
    s.key, s.value = kv[..., :s.nope], kv[..., s.nope:]
    s.rope_key = torch.randn((n, ROPE), generator=g, device=dev).to(s.dtype)
    s.q = (1.5 * torch.randn((s.nnz, s.heads, s.nope + ROPE), generator=g, device=dev)).to(s.dtype)
    s.scale = 1 / math.sqrt(s.nope + ROPE)
    return s


def run(s):
    if own:
        from paceserve_amd.kv_transfer import latent, rope, tables
        if s.kind == "tables":
            return tables.build_tables(s.page_table, s.seq_lens, s.P, s.qo_indptr, s.nnz)._asdict()
        if s.kind == "rotate":
            q, k = rope.norm_rotate(s.q, s.k, s.positions, s.table, s.q_weight, s.k_weight, eps=EPS,
                                    interleaved=s.interleaved)
            return {"q": q, "k": k}
        if s.kind == "write":
            q = rope.append_paged_kv_cache_rope(s.q, s.k, s.v, s.positions, s.slot_mapping, s.cache, s.table, s.q_weight,
                                                s.k_weight, eps=EPS, interleaved=s.interleaved)
            return {"q": q, "cache": _typed(s)}
        if s.kind == "latent":
            latent.append_paged_latent_cache(s.latent, s.rope_key, s.positions, s.slot_mapping, s.cache, s.table,
                                             s.weight, eps=EPS, interleaved=s.interleaved)
            return s.cache
        if s.kind == "absorbed":
            out, lse = latent.paged_latent_attention(s.q, s.cache, s.kv_indices, s.kv_indptr, s.last, s.qo_indptr,
                                                     sm_scale=s.scale, max_q_len=s.max_new, tree_mask=s.mask,
                                                     return_lse=True)
        else:
            out, lse = latent.latent_prompt_attention(s.q, s.key, s.rope_key, s.value, s.qo_indptr, s.kv_indptr,
                                                      sm_scale=s.scale, max_q_len=s.max_new, return_lse=True)
        return {"out": out, "lse": lse}
    if s.kind == "tables":
        return _tables(s)
    if s.kind == "rotate":
        return {"q": _norm_rotate(s, s.q, s.q_weight).to(s.dtype), "k": _norm_rotate(s, s.k, s.k_weight).to(s.dtype)}
    if s.kind == "write":
        return _write(s)
    if s.kind == "latent":
        return _latent(s)
    return _absorbed(s) if s.kind == "absorbed" else _prompt(s)


# ---------------------------------------------------------------- 64 bits

def _turned64(x, weight, positions, table, interleaved):
    """Rows [n, heads, D] normalised and turned, as complex numbers."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * weight.double()
    r = table.shape[1]
    turn = torch.complex(*(table[positions.long()].double().split(r // 2, 1)))[:, None, :]
    head = x[..., :r]
    pairs = head.unflatten(-1, (r // 2, 2)) if interleaved else head.unflatten(-1, (2, r // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    z = z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)
    return torch.cat([z, x[..., r:]], -1)


def _written64(s, kv):
    """The cache's outputs after rows kv [n, 2, H, D] (float64) went into their slots."""
    page, slot = s.slot_mapping // s.P, s.slot_mapping % s.P
    if s.cache.dtype != torch.uint8:
        out = s.cache.double()
        out[page, :, slot] = kv
        return out
    data, byte = _halves(s.cache, s.D)
    el, sc = data.view(torch.float8_e4m3fn).double(), torch.exp2(byte.double() - 127)
    m, e = torch.frexp(kv.unflatten(-1, (-1, BLOCK)).abs().amax(-1) / 448)                 # m in [0.5, 1)
    e = torch.where(m == 0, -117.0, torch.where(m > 0.5, e, e - 1).double()).clamp(-117, 127)
    y = (kv.unflatten(-1, (-1, BLOCK)) * torch.exp2(-e).unsqueeze(-1)).flatten(-2)
    step = torch.exp2((torch.frexp(y.abs())[1].double() - 1).clamp(min=-6) - 3)
    el[page, :, slot], sc[page, :, slot] = torch.round(y / step) * step, torch.exp2(e)
    return {"elements": el, "scales": sc}


def _attention64(q, k, v, scale, hidden):
    """One request and head: q [t, D], k [n, D], v [n, Dv] in float64."""
    x = (q @ k.T * scale).masked_fill(hidden, -math.inf)
    return torch.softmax(x, -1) @ v, torch.logsumexp(x, -1)


def exact(case, seed):
    if case["kind"] == "tables" or work(case)["flops"] > 2e12:
        return None
    s = prepare(case, seed)
    if s.kind in ("rotate", "write"):
        q, k = (_turned64(x, w, s.positions, s.table, s.interleaved) for x, w in ((s.q, s.q_weight), (s.k, s.k_weight)))
        if s.kind == "rotate":
            return {"q": q, "k": k}
        return {"q": q, "cache": _written64(s, torch.stack([k, s.v.double()], 1))}
    if s.kind == "latent":
        c = s.latent.double()
        c = c / torch.sqrt((c * c).sum(-1, keepdim=True) / s.L + EPS) * s.weight.double()
        k = _turned64(s.rope_key[:, None], None, s.positions, s.table, s.interleaved)[:, 0]
        out = s.cache.double()
        out[s.slot_mapping // s.P, s.slot_mapping % s.P] = torch.cat([c, k], 1)
        return out
    qo, ip = s.qo_indptr.tolist(), s.kv_indptr.tolist()
    width = s.L if s.kind == "absorbed" else s.nope
    out = torch.zeros((s.nnz, s.heads, width), dtype=torch.float64, device=s.dev)
    lse = torch.zeros((s.nnz, s.heads), dtype=torch.float64, device=s.dev)
    last = s.last.tolist() if s.kind == "absorbed" else None
    for b in range(s.requests):
        at, t = slice(qo[b], qo[b + 1]), qo[b + 1] - qo[b]
        n = (ip[b + 1] - ip[b] - 1) * s.P + last[b] if last else ip[b + 1] - ip[b]
        hidden = torch.zeros((t, n), dtype=torch.bool, device=s.dev)
        tail = torch.ones((t, t), dtype=torch.bool, device=s.dev).triu(1)
        if last and s.mask is not None:
            tail = ((s.mask[at] >> torch.arange(64, device=s.dev)) & 1)[:, :t] == 0
        hidden[:, n - t:] = tail
        if last:
            kv = s.cache[s.kv_indices[ip[b]:ip[b + 1]].long()].flatten(0, 1)[:n].double()
            o, e = _attention64(s.q[at].double().flatten(0, 1), kv, kv[:, :s.L], s.scale,
                                hidden.repeat_interleave(s.heads, 0))
            out[at], lse[at] = o.unflatten(0, (t, s.heads)), e.unflatten(0, (t, s.heads))
            continue
        keys = slice(ip[b], ip[b + 1])
        for h in range(s.heads):
            k = torch.cat([s.key[keys, h], s.rope_key[keys]], 1).double()
            out[at, h], lse[at, h] = _attention64(s.q[at, h].double(), k, s.value[keys, h].double(), s.scale, hidden)
    return {"out": out, "lse": lse}
