"""What the library refuses on the host of the calls around a paged cache at the ends
of their ranges (no GPU)."""
import pytest

from paceserve_amd import _native

LIB = _native.load()
EINVAL, ERANGE = _native.PACE_KV_EINVAL, _native.PACE_KV_ERANGE


def refused(code, args, want, msg):
    assert code == want, (args, code)
    assert msg in LIB.pace_kv_last_error().decode()


def append_packed(q=0x1000, q_token=4096, q_head=256, heads=8, q_out=0x2000, out_token=4096, out_head=256, k=0x3000,
                  v=0x4000, k_heads=1, D=128, nnz=3, slots=0x100, r=128, eps=1e-6, cache=0x5000, fmt=1, pages=4, P=1):
    return LIB.pace_kv_append_rope_packed(q, q_token, q_head, heads, q_out, out_token, out_head, None, k, 1024, 256, None, v,
                                          1024, 256, k_heads, 0, D, nnz, 0x100, slots, 0x100, 9, r, 0, eps, cache, fmt,
                                          pages, P, None, None)


@pytest.mark.parametrize("args,code,msg", [
    (dict(q=None), EINVAL, "NULL"), (dict(cache=None), EINVAL, "NULL"), (dict(slots=None), EINVAL, "NULL"),
    (dict(cache=0x5008), EINVAL, "16-byte"), (dict(slots=0x104), EINVAL, "8-byte"), (dict(fmt=3), EINVAL, "format"),
    (dict(D=80, r=64), EINVAL, "64"), (dict(r=32), EINVAL, "64"), (dict(k_heads=0), EINVAL, "KV heads"),
    (dict(P=0), EINVAL, "page size"), (dict(pages=-1), EINVAL, "pages"), (dict(eps=-1.0), EINVAL, "eps"),
    (dict(out_head=128), EINVAL, "overlap"), (dict(P=(1 << 31) - 1, k_heads=1 << 20), ERANGE, "2^36")])
def test_packed_pages_refuse_what_others_do(args, code, msg):
    refused(append_packed(**args), args, code, msg)
    assert append_packed(nnz=0) == 0
