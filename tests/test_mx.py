"""The quantised cache's format and the refusals of its calls (no GPU): row
widths, the 64-bit oracle against torch's own e4m3 conversion, and argument
errors that the library finds on the host."""
import numpy as np
import pytest
import torch

from oracle import mx_oracle as mo
from paceserve_amd import _native
from paceserve_amd.kv_transfer import mx

LIB = _native.load()
EINVAL, ERANGE = _native.PACE_KV_EINVAL, _native.PACE_KV_ERANGE


def test_row_widths():
    assert mx.row_width(128, "mxfp8") == 132 and mx.row_width(128, "mxfp4") == 68 and mx.row_width(32, "mxfp4") == 17
    for D, fmt in ((0, "mxfp8"), (100, "mxfp8"), (-32, "mxfp4"), (128, "fp8")):
        with pytest.raises(ValueError):
            mx.row_width(D, fmt)
    for D in range(32, 1056, 32):                       # a width names its format
        assert mx._format_of(mx.row_width(D, "mxfp8"), D) == _native.MXFP8
        assert mx._format_of(mx.row_width(D, "mxfp4"), D) == _native.MXFP4
    with pytest.raises(ValueError, match="no format"):
        mx._format_of(128, 128)


def test_elements_and_scales_are_views():
    c = mx.empty_cache(3, 4, 2, 64, "mxfp4", device="cpu")
    e, s = mx.elements_and_scales(c, 64)
    assert e.shape == (3, 2, 4, 2, 32) and s.shape == (3, 2, 4, 2, 2)
    e.fill_(7), s.fill_(9)
    flat = c.view(3, 2, -1)
    assert (flat[:, :, :256] == 7).all() and (flat[:, :, 256:] == 9).all() and flat.shape[2] == 272


def test_oracle_rounds_as_torch_does():
    rng = np.random.default_rng(5)
    x = np.concatenate([rng.standard_normal(1 << 16) * 60, np.linspace(-448, 448, 1 << 14),
                        rng.standard_normal(1 << 14) * 2.0 ** -8])
    x = x.astype(np.float32).astype(np.float64).reshape(-1, 32)
    x[:, 0] = 448                                        # every scale is 1
    codes, byte = mo.quantize(x, "mxfp8")
    assert (byte == 127).all()
    want = torch.from_numpy(x).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(codes, want)
    back = mo.values(codes, byte, "mxfp8")
    assert np.array_equal(back, torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy())


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_oracle_scale_is_the_smallest_that_holds(fmt):
    top = mo.TOP[fmt]
    for a, e in ((top, 0), (np.nextafter(top, 1e9), 1), (top / 2, -1), (0.0, -117), (1e-45, -117),
                 (top * 2.0 ** -118, -117), (3.38e38, 120 if fmt == "mxfp8" else 126)):
        x = np.zeros((1, 32))
        x[0, 7] = -a
        assert mo.quantize(x, fmt)[1][0, 0] == e + 127, a
    for bad in (np.inf, -np.inf, np.nan):
        x = np.ones((1, 64))
        x[0, 40] = bad
        codes, byte = mo.quantize(x, fmt)
        assert byte[0, 1] == 255 and byte[0, 0] < 255 and not codes[0, 32:].any()
        back = mo.values(mo.pack(codes, fmt), byte, fmt)
        assert np.isnan(back[0, 32:]).all() and (back[0, :32] == 1).all()


def test_oracle_ties_go_to_the_even_code():
    x = np.array([[6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5] + [0.0] * 24])
    assert mo.quantize(x, "mxfp4")[0][0, :8].tolist() == [7, 0, 2, 2, 4, 4, 6, 6]


def _append(nnz=1, type=0, stride=2048, batch=1, fmt=1, pages=4, page_size=16, row=1024, key=0x1000, cache=0x2000,
            indptr=0x100, fused=False):
    if fused:
        return LIB.pace_kv_append_mx_indptr(key, 0x1000, type, stride, nnz, 0x100, batch, cache, fmt, pages, 0x100, 4,
                                            indptr, 0x100, page_size, row, None, None)
    return LIB.pace_kv_append_mx(key, 0x1000, type, stride, nnz, 0x100, 0x100, batch, cache, fmt, pages, 0x100, 4,
                                 indptr, page_size, row, None, None)


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("args,code,msg", [
    (dict(nnz=-1), EINVAL, "negative"), (dict(type=3), EINVAL, "element type"), (dict(fmt=0), EINVAL, "format"),
    (dict(fmt=3), EINVAL, "format"), (dict(key=None), EINVAL, "NULL"), (dict(page_size=0), EINVAL, "page_size"),
    (dict(row=1000), EINVAL, "blocks of 32"), (dict(row=0), EINVAL, "blocks of 32"),
    (dict(page_size=1, row=96, stride=192), EINVAL, "multiple of 16"),
    (dict(stride=2032), EINVAL, "token stride"), (dict(stride=2056), EINVAL, "token stride"),
    (dict(type=2), EINVAL, "token stride"), (dict(key=0x1008), EINVAL, "aligned"),
    (dict(cache=0x2004), EINVAL, "aligned"), (dict(pages=1 << 31), ERANGE, "pages"),
    (dict(nnz=1 << 24), ERANGE, "tokens"), (dict(nnz=1 << 31), ERANGE, "tokens"),
    (dict(row=1 << 31, stride=1 << 33), ERANGE, "row too large")])
def test_append_refuses(fused, args, code, msg):
    assert _append(fused=fused, **args) == code
    assert msg in LIB.pace_kv_last_error().decode()


def test_append_of_nothing_is_a_no_op():
    assert _append(nnz=0, key=None) == 0 and _append(nnz=0, key=None, fused=True) == 0
    assert _append(nnz=1, batch=0, fused=True) == EINVAL


def _convert(down=True, layers=1, pages=2, type=0, fmt=1, half=16384, src=0x10000, dst=0x20000, ids=0x100, pool=9):
    s, d = _native.pointer_array([src] * max(layers, 1)), _native.pointer_array([dst] * max(layers, 1))
    if down:
        return LIB.pace_kv_quantize_pages(s, pool, ids, type, d, 9, 0x100, fmt, layers, pages, half, None, None)
    return LIB.pace_kv_dequantize_pages(s, pool, ids, fmt, d, 9, 0x100, type, layers, pages, half, None, None)


@pytest.mark.parametrize("down", [True, False])
@pytest.mark.parametrize("args,code,msg", [
    (dict(layers=-1), EINVAL, "negative"), (dict(pages=-1), EINVAL, "negative"), (dict(pool=-1), EINVAL, "negative"),
    (dict(type=7), EINVAL, "element type"), (dict(fmt=0), EINVAL, "format"), (dict(ids=None), EINVAL, "NULL"),
    (dict(src=0), EINVAL, "NULL"), (dict(half=0), EINVAL, "blocks of 32"), (dict(half=16000 + 16), EINVAL, "blocks"),
    (dict(half=96), EINVAL, "multiple of 16"), (dict(ids=0x102), EINVAL, "4-byte"),
    (dict(src=0x10008), EINVAL, "16-byte"), (dict(dst=0x20004), EINVAL, "16-byte"),
    (dict(pool=1 << 31), ERANGE, "pages"), (dict(half=1 << 41), ERANGE, "page too large")])
def test_conversion_refuses(down, args, code, msg):
    assert _convert(down, **args) == code
    assert msg in LIB.pace_kv_last_error().decode()


def test_conversion_of_nothing_is_a_no_op():
    for down in (True, False):
        assert _convert(down, layers=0) == 0 and _convert(down, pages=0) == 0


def test_python_checks_name_what_is_wrong():
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="uint8 device tensor"):
        mx.append_paged_kv_cache_mx_indptr(k, k, i, mx.empty_cache(2, 4, 2, 64, "mxfp8", device="cpu"), i, i, i)
    with pytest.raises(ValueError, match="device tensors"):
        mx.quantize_pages([torch.zeros(2, 2, 4, 2, 64)], [0], [mx.empty_cache(2, 4, 2, 64, "mxfp8", device="cpu")], [0])
