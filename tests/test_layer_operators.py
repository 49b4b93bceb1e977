"""What the library refuses on the host of the calls around a paged cache (its
tables, norms with rotation, latent attention), the sizes of their workspaces,
tensors that want gradients, and the oracle of rotated rows (no GPU)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import rope_oracle as ro
from paceserve_amd import _native
from paceserve_amd.kv_transfer import latent, ops, rope, tables

LIB = _native.load()
EINVAL, ERANGE = _native.PACE_KV_EINVAL, _native.PACE_KV_ERANGE


def refused(call, args, code, msg):
    assert call(**args) == code
    assert msg in LIB.pace_kv_last_error().decode()


def build(table=0x100, stride=8, width=8, lens=0x100, batch=2, P=16, indptr=0x100, nnz=4, idx=0x100, num_indices=6,
          kv=0x100, last=0x100, pos=0x100, slots=0x100):
    return LIB.pace_kv_build_tables(table, stride, width, lens, batch, P, indptr, nnz, idx, num_indices, kv, last, pos,
                                    slots, None, None)


@pytest.mark.parametrize("args,code,msg", [
    (dict(batch=-1), EINVAL, "negative"), (dict(width=-1), EINVAL, "negative"), (dict(nnz=-1), EINVAL, "negative"),
    (dict(num_indices=-1), EINVAL, "negative"), (dict(P=0), EINVAL, "no tokens"), (dict(nnz=1 << 31), ERANGE, "2^31"),
    (dict(num_indices=1 << 31), ERANGE, "2^31"), (dict(batch=1 << 16, width=1 << 16), ERANGE, "2^31"),
    (dict(table=None), EINVAL, "NULL"), (dict(lens=None), EINVAL, "NULL"), (dict(idx=None), EINVAL, "NULL"),
    (dict(kv=None), EINVAL, "NULL"), (dict(last=None), EINVAL, "NULL"), (dict(pos=None), EINVAL, "NULL"),
    (dict(slots=None), EINVAL, "NULL"), (dict(stride=7), EINVAL, "overlap"),
    (dict(indptr=None, nnz=1), EINVAL, "one token")])
def test_tables_refuse(args, code, msg):
    refused(build, args, code, msg)


def turn(q=0x1000, q_token=4096, q_head=256, heads=8, q_out=0x2000, out_token=4096, out_head=256, qw=None, k=0x3000,
         k_head=256, k_heads=2, k_out=0x4000, kw=None, type=0, D=128, nnz=3, pos=0x100, table=0x100, rows=9, r=128,
         eps=1e-6):
    return LIB.pace_kv_norm_rotate(q, q_token, q_head, heads, q_out, out_token, out_head, qw, k, 1024, k_head, k_heads,
                                   k_out, 1024, 256, kw, type, D, nnz, pos, table, rows, r, 0, eps, None, None)


SHARED = [
    (dict(D=100), EINVAL, "multiples of 16"), (dict(D=0), EINVAL, "multiples of 16"), (dict(D=2048), EINVAL, "1024"),
    (dict(r=0), EINVAL, "rotary_dim"), (dict(r=144), EINVAL, "rotary_dim"), (dict(r=24), EINVAL, "rotary_dim"),
    (dict(heads=-1), EINVAL, "heads"), (dict(heads=1 << 21), EINVAL, "heads"), (dict(nnz=-1), EINVAL, "negative"),
    (dict(rows=-1), EINVAL, "negative"), (dict(type=2), EINVAL, "bfloat16 or float16"), (dict(eps=-1.0), EINVAL, "eps"),
    (dict(eps=math.nan), EINVAL, "eps"), (dict(eps=math.inf), EINVAL, "eps"), (dict(pos=None), EINVAL, "NULL"),
    (dict(table=None), EINVAL, "NULL"), (dict(table=0x108), EINVAL, "16-byte"), (dict(q=None), EINVAL, "NULL"),
    (dict(q_out=None), EINVAL, "NULL"), (dict(k=None), EINVAL, "NULL"), (dict(q=0x1008), EINVAL, "16 bytes"),
    (dict(q_token=4104), EINVAL, "16 bytes"), (dict(out_head=264), EINVAL, "16 bytes"), (dict(qw=0x108), EINVAL, "16 bytes"),
    (dict(kw=0x108), EINVAL, "16 bytes"), (dict(out_head=128), EINVAL, "overlap"), (dict(out_head=-240), EINVAL, "overlap"),
    (dict(out_token=0), EINVAL, "overlap"), (dict(out_token=240), EINVAL, "overlap")]


@pytest.mark.parametrize("args,code,msg", SHARED + [(dict(k_out=None), EINVAL, "NULL"), (dict(k_out=0x4008), EINVAL, "16 bytes")])
def test_norm_rotate_refuses(args, code, msg):
    refused(turn, args, code, msg)


def append(q=0x1000, q_token=4096, q_head=256, heads=8, q_out=0x2000, out_token=4096, out_head=256, qw=None, k=0x3000,
           kw=None, v=0x4000, v_token=1024, k_heads=2, type=0, D=128, nnz=3, pos=0x100, slots=0x100, table=0x100, rows=9,
           r=128, eps=1e-6, cache=0x5000, fmt=0, pages=4, P=16):
    return LIB.pace_kv_append_rope(q, q_token, q_head, heads, q_out, out_token, out_head, qw, k, 1024, 256, kw, v, v_token,
                                   256, k_heads, type, D, nnz, pos, slots, table, rows, r, 0, eps, cache, fmt, pages, P,
                                   None, None)


@pytest.mark.parametrize("args,code,msg", SHARED + [
    (dict(v=None), EINVAL, "NULL"), (dict(v_token=1032), EINVAL, "16 bytes"), (dict(k_heads=0), EINVAL, "KV heads"),
    (dict(fmt=3), EINVAL, "format"), (dict(fmt=1, D=80, r=64), EINVAL, "64"), (dict(fmt=2, r=32), EINVAL, "64"),
    (dict(pages=-1), EINVAL, "pages"), (dict(pages=1 << 31), EINVAL, "pages"), (dict(P=0), EINVAL, "page size"),
    (dict(slots=None), EINVAL, "NULL"), (dict(slots=0x104), EINVAL, "8-byte"), (dict(cache=None), EINVAL, "NULL"),
    (dict(cache=0x5008), EINVAL, "16-byte"), (dict(P=(1 << 31) - 1, k_heads=1 << 20), ERANGE, "2^36"),
    (dict(fmt=1, k_heads=1, D=64, r=64, P=1, q_head=128, out_head=128), EINVAL, "multiple of 16")])
def test_append_rope_refuses(args, code, msg):
    refused(append, args, code, msg)


def append_latent(x=0x1000, x_token=1152, k=0x2000, k_token=1152, w=None, type=0, L=512, nnz=3, pos=0x100, slots=0x100,
                  table=0x100, rows=9, eps=1e-6, cache=0x5000, pages=4, P=16):
    return LIB.pace_kv_append_latent(x, x_token, k, k_token, w, type, L, nnz, pos, slots, table, rows, 0, eps, cache, pages,
                                     P, None, None)


@pytest.mark.parametrize("args,code,msg", [
    (dict(L=128), EINVAL, "256 or 512"), (dict(type=2), EINVAL, "bfloat16 or float16"), (dict(nnz=-1), EINVAL, "negative"),
    (dict(rows=-1), EINVAL, "negative"), (dict(eps=math.nan), EINVAL, "eps"), (dict(pos=None), EINVAL, "NULL"),
    (dict(table=None), EINVAL, "NULL"), (dict(table=0x104), EINVAL, "16-byte"), (dict(x=None), EINVAL, "NULL"),
    (dict(k=None), EINVAL, "NULL"), (dict(slots=None), EINVAL, "NULL"), (dict(cache=None), EINVAL, "NULL"),
    (dict(x=0x1008), EINVAL, "16 bytes"), (dict(x_token=1160), EINVAL, "16 bytes"), (dict(k=0x2002), EINVAL, "16 bytes"),
    (dict(k_token=130), EINVAL, "16 bytes"), (dict(w=0x108), EINVAL, "16 bytes"), (dict(cache=0x5004), EINVAL, "16 bytes"),
    (dict(slots=0x104), EINVAL, "slot_mapping"), (dict(pages=-1), EINVAL, "pages"), (dict(P=0), EINVAL, "page size"),
    (dict(nnz=1 << 40), ERANGE, "too many")])
def test_append_latent_refuses(args, code, msg):
    refused(append_latent, args, code, msg)


def absorbed(q=0x1000, stride=16 * 1152, type=0, nnz=8, qo=0x100, batch=2, heads=16, L=512, cache=0x2000, pages=9, P=16,
             idx=0x100, num_indices=6, indptr=0x100, last=0x100, max_q=4, mask=None, words=0, scale=0.1, out=0x3000,
             out_stride=16 * 1024, space=None, size=0):
    return LIB.pace_kv_latent_attention(q, stride, type, nnz, qo, batch, heads, L, cache, pages, P, idx, num_indices, indptr,
                                        last, max_q, mask, words, scale, out, out_stride, None, space, size, None, None)


@pytest.mark.parametrize("args,code,msg", [
    (dict(nnz=-1), EINVAL, "negative"), (dict(batch=-1), EINVAL, "positive"), (dict(heads=0), EINVAL, "positive"),
    (dict(max_q=0), EINVAL, "positive"), (dict(P=0), EINVAL, "positive"), (dict(num_indices=-1), EINVAL, "positive"),
    (dict(L=128), EINVAL, "256 or 512"), (dict(type=2), EINVAL, "bfloat16 or float16"), (dict(pages=-1), ERANGE, "pages"),
    (dict(pages=1 << 31), ERANGE, "pages"), (dict(scale=math.nan), EINVAL, "scale"), (dict(scale=math.inf), EINVAL, "scale"),
    (dict(scale=3e38), EINVAL, "scale"), (dict(q=None), EINVAL, "NULL"), (dict(cache=None), EINVAL, "NULL"),
    (dict(idx=None), EINVAL, "NULL"), (dict(indptr=None), EINVAL, "NULL"), (dict(last=None), EINVAL, "NULL"),
    (dict(out=None), EINVAL, "NULL"), (dict(qo=None), EINVAL, "one token"), (dict(mask=0x100), EINVAL, "mask"),
    (dict(mask=0x100, words=1, max_q=65), EINVAL, "mask"), (dict(mask=0x104, words=1), EINVAL, "8-byte"),
    (dict(stride=16 * 1152 - 16), EINVAL, "strides"), (dict(stride=16 * 1152 + 8), EINVAL, "strides"),
    (dict(out_stride=16 * 1024 - 16), EINVAL, "strides"), (dict(q=0x1008), EINVAL, "aligned"),
    (dict(cache=0x2008), EINVAL, "aligned"), (dict(out=0x3004), EINVAL, "aligned"), (dict(pages=1 << 22), ERANGE, "64 GiB"),
    (dict(num_indices=1 << 27), ERANGE, "tokens"), (dict(nnz=1 << 20), ERANGE, "query rows"),
    (dict(batch=1 << 24), ERANGE, "too many"), (dict(max_q=1 << 26), ERANGE, "rows"),
    (dict(num_indices=4096), EINVAL, "workspace"), (dict(num_indices=4096, space=0x1000, size=64), EINVAL, "workspace"),
    (dict(num_indices=4096, space=0x1008, size=1 << 40), EINVAL, "workspace")])
def test_latent_attention_refuses(args, code, msg):
    refused(absorbed, args, code, msg)


def prompt(q=0x1000, q_token=16 * 384, q_head=384, k=0x2000, k_token=16 * 512, rk=0x3000, r_token=128, v=0x4000,
           v_token=16 * 512, type=0, heads=16, D=128, nnz=8, keys=40, qo=0x100, kv=0x100, batch=2, max_q=8, scale=0.1,
           out=0x5000, o_token=16 * 256, o_head=256, space=None, size=0):
    return LIB.pace_kv_prompt_attention(q, q_token, q_head, k, k_token, 512, rk, r_token, v, v_token, 512, type, heads, D,
                                        nnz, keys, qo, kv, batch, max_q, scale, 1, out, o_token, o_head, None, space, size,
                                        None, None)


@pytest.mark.parametrize("args,code,msg", [
    (dict(nnz=-1), EINVAL, "positive"), (dict(keys=-1), EINVAL, "positive"), (dict(batch=-1), EINVAL, "positive"),
    (dict(heads=0), EINVAL, "positive"), (dict(max_q=0), EINVAL, "positive"), (dict(D=96), EINVAL, "64 or 128"),
    (dict(type=2), EINVAL, "bfloat16 or float16"), (dict(scale=math.nan), EINVAL, "scale"), (dict(q=None), EINVAL, "NULL"),
    (dict(k=None), EINVAL, "NULL"), (dict(rk=None), EINVAL, "NULL"), (dict(v=None), EINVAL, "NULL"),
    (dict(out=None), EINVAL, "NULL"), (dict(qo=None), EINVAL, "NULL"), (dict(kv=None), EINVAL, "NULL"),
    (dict(q=0x1008), EINVAL, "16 bytes"), (dict(k_token=8), EINVAL, "16 bytes"), (dict(r_token=130), EINVAL, "16 bytes"),
    (dict(out=0x5002), EINVAL, "16 bytes"), (dict(q_head=390), EINVAL, "16 bytes"),
    (dict(k_token=1 << 26), EINVAL, "2^26"), (dict(v_token=-8192), EINVAL, "2^26"), (dict(nnz=1 << 31), ERANGE, "2^30"),
    (dict(keys=1 << 31), ERANGE, "2^30"), (dict(nnz=1 << 26), ERANGE, "too many"),
    (dict(o_token=0), EINVAL, "overlap"), (dict(o_token=240), EINVAL, "overlap"), (dict(o_head=128), EINVAL, "overlap"),
    (dict(heads=(1 << 20) + 1), ERANGE, "too many"), (dict(keys=60000), EINVAL, "workspace"),
    (dict(keys=60000, space=0x1000, size=64), EINVAL, "workspace"),
    (dict(keys=60000, space=0x1008, size=1 << 40), EINVAL, "workspace")])
def test_prompt_attention_refuses(args, code, msg):
    refused(prompt, args, code, msg)


def test_nothing_to_do():
    assert turn(nnz=0) == 0 and turn(heads=0, k_heads=0) == 0
    assert append(nnz=0) == 0 and append_latent(nnz=0) == 0
    assert absorbed(nnz=0) == 0 and absorbed(batch=0) == 0
    assert prompt(nnz=0) == 0 and prompt(batch=0) == 0


def test_workspaces():
    out = ctypes.c_int64(-1)

    def latent_space(batch, heads, L, max_q, num_indices, P, to=ctypes.byref(out)):
        return LIB.pace_kv_latent_attention_workspace(batch, heads, L, max_q, num_indices, P, to)

    def prompt_space(nnz, keys, batch, heads, D, to=ctypes.byref(out)):
        return LIB.pace_kv_prompt_attention_workspace(nnz, keys, batch, heads, D, 1, to)

    assert latent_space(2, 16, 512, 1, 2, 16) == 0 and out.value == 0
    assert latent_space(1, 16, 512, 1, 4096, 16) == 0 and out.value > 0
    # as many parts as whole chunks fit the pages, twice: a part is a tile of rows of L + 2 floats
    assert out.value % (16 * 514 * 4) == 0 and out.value <= 2 * 4096 * 16 * 514 * 4
    assert latent_space(1, 16, 512, 1, 4096, 16, None) == EINVAL and latent_space(1, 16, 100, 1, 4096, 16) == EINVAL
    # products past 64 bits
    for sizes in ((1016, 1 << 30, 512, (1 << 30) - 1, 0, 16), (1, 1, 512, 1, 1 << 60, 16), (1, 1, 512, 1, (1 << 62) + 1, 4),
                  ((1 << 31) - 1, 1, 512, 1, 0, 16)):
        assert latent_space(*sizes) == ERANGE
    assert prompt_space(64, 64, 1, 16, 128) == 0 and out.value == 0
    assert prompt_space(64, 60000, 1, 16, 128) == 0 and out.value > 0 and out.value % (64 * 16 * 130 * 4) == 0
    assert prompt_space(0, 0, 0, 16, 128) == 0 and out.value == 0
    assert prompt_space(64, 64, 1, 16, 128, None) == EINVAL and prompt_space(64, 64, 1, 16, 32) == EINVAL
    assert prompt_space(1 << 30, 1 << 30, (1 << 31) - 1, 1, 128) == ERANGE


def test_tensors_that_want_gradients_are_refused():
    x, rows = torch.zeros(2, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 512, dtype=torch.bfloat16)
    i, s = torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    t, cache = torch.zeros(4, 64), torch.zeros(1, 2, 16, 2, 64, dtype=torch.bfloat16)
    kept = torch.zeros(1, 16, 576, dtype=torch.bfloat16)
    q = torch.zeros(2, 4, 576, dtype=torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16, requires_grad=True)
    calls = [
        lambda g: rope.norm_rotate(g(x), x, i, t), lambda g: rope.norm_rotate(x, g(x), i, t),
        lambda g: rope.norm_rotate(x, x, i, t, w if g is grad else None),
        lambda g: rope.append_paged_kv_cache_rope(x, x, g(x), i, s, cache, t),
        lambda g: rope.append_paged_kv_cache_rope(x, x, x, i, s, g(cache), t),
        lambda g: latent.append_paged_latent_cache(g(rows), x[:, 0], i, s, kept, t),
        lambda g: latent.append_paged_latent_cache(rows, x[:, 0], i, s, g(kept), t),
        lambda g: latent.paged_latent_attention(g(q), kept, i, i, i, sm_scale=1.0),
        lambda g: latent.paged_latent_attention(q, g(kept), i, i, i, sm_scale=1.0),
        lambda g: latent.latent_prompt_attention(g(q[..., :128]), x, x[:, 0], x, i, i),
        lambda g: latent.latent_prompt_attention(q[..., :128], x, x[:, 0], g(x), i, i)]

    def grad(y):
        return y.clone().requires_grad_()

    for call in calls:
        with pytest.raises(ValueError, match="no backward"):
            call(grad)
        with torch.no_grad(), pytest.raises(ValueError) as e:              # the next thing wrong: no device tensors
            call(grad)
        assert "no backward" not in str(e.value)
        with pytest.raises(ValueError) as e:
            call(lambda y: y)
        assert "no backward" not in str(e.value)


def test_host_tensors_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        tables.build_tables(torch.zeros(2, 4, dtype=torch.int32), i, 16, num_indices=4)
    with pytest.raises(ValueError):
        latent.empty_cache(1, 16, 100, device=torch.device("cpu"))
    with pytest.raises(ValueError, match="latent"):
        ops.PagedPool([torch.zeros(4, 2, 16, 64)])                          # neither form
    with pytest.raises(ValueError, match="device"):
        ops.PagedPool([latent.empty_cache(2, 16, 512, device=torch.device("cpu"))])


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_oracle_turns_complex_numbers(interleaved):
    """Columns (a, b) times (cos + i sin) of position and frequency; the rest stays."""
    rng = np.random.default_rng(0)
    x, w = rng.standard_normal((3, 32)), rng.standard_normal(32)
    angle = 7 * 10000.0 ** (-np.arange(8) / 8)
    y, size = ro.turned(x, w, 1e-6, np.concatenate([np.cos(angle), np.sin(angle)]), interleaved)
    z = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + 1e-6) * w
    head = z[:, :16].reshape(3, 8, 2) if interleaved else z[:, :16].reshape(3, 2, 8).transpose(0, 2, 1)
    want = (head[..., 0] + 1j * head[..., 1]) * np.exp(1j * angle)
    got = y[:, :16].reshape(3, 8, 2) if interleaved else y[:, :16].reshape(3, 2, 8).transpose(0, 2, 1)
    # ten operations of 2^-53 each on numbers below 8
    assert np.abs(got[..., 0] - want.real).max() < 1e-13 and np.abs(got[..., 1] - want.imag).max() < 1e-13
    assert np.array_equal(y[:, 16:], z[:, 16:]) and (size >= np.abs(y) - 1e-13).all()
