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


def turn(q_token=4096, heads=8, out_token=4096, out_head=256, k_out_token=1024, k_out_head=256, D=128, nnz=3, r=128):
    return LIB.pace_kv_norm_rotate(0x1000, q_token, 256, heads, 0x2000, out_token, out_head, None, 0x3000, 1024, 256, 2, 0x4000,
                                   k_out_token, k_out_head, None, 0, D, nnz, 0x100, 0x100, 9, r, 0, 1e-6, None, None)


def prompt(o_token=16 * 256, o_head=256, heads=16, nnz=8):
    return LIB.pace_kv_prompt_attention(0x1000, 16 * 384, 384, 0x2000, 16 * 512, 512, 0x3000, 128, 0x4000, 16 * 512, 512, 0,
                                        heads, 128, nnz, 40, 0x100, 0x100, 2, 8, 0.1, 1, 0x5000, o_token, o_head, None, None, 0,
                                        None, None)


@pytest.mark.parametrize("token,head", [
    (256, 256), (256 * 7, 256), (-256, 256), (256, -256), (512, 768), (768, 512), (256 * 8 - 16, 256), (256, 256 * 3 - 16),
    (384, 256), (256, 384), (1 << 62, 1 << 62), (256 * 5 - 16, 512)])
def test_rows_of_one_token_and_another_that_overlap(token, head):
    """Each of the strides alone keeps rows of 256 bytes apart, both together do not."""
    args = dict(token=token, head=head)
    refused(turn(out_token=token, out_head=head, nnz=9), args, EINVAL, "overlap")
    refused(append_packed(out_token=token, out_head=head, nnz=9), args, EINVAL, "overlap")
    refused(prompt(o_token=token, o_head=head, nnz=9), args, EINVAL, "overlap")
    if token == head:
        refused(turn(k_out_token=token, k_out_head=head), args, EINVAL, "overlap")


def append_latent(nnz, L=512):
    return LIB.pace_kv_append_latent(0x1000, 1152, 0x2000, 1152, None, 0, L, nnz, 0x100, 0x100, 0x100, 9, 0, 1e-6, 0x5000, 4,
                                     16, None, None)


@pytest.mark.parametrize("nnz", [1 << 26, (1 << 26) - 3, 1 << 31, 1 << 40, (1 << 63) - 1])
def test_launches_of_two_to_the_32_threads(nnz):
    """Threads of a launch are counted in 32 bits: 2^24 workgroups of 256 are one too many."""
    refused(turn(nnz=nnz), nnz, ERANGE, "too many tokens")
    refused(append_packed(nnz=nnz), nnz, ERANGE, "too many tokens")
    # eight rows of 512 columns a workgroup, sixteen of 256
    for L, rows in ((512, 8), (256, 16)):
        refused(append_latent(min(nnz * rows // 4, (1 << 63) - 1), L), nnz, ERANGE, "too many tokens")
