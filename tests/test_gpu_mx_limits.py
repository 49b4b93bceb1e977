"""The quantised format at the low end of its types: blocks of numbers near and
below the smallest scale, subnormal ones among them, byte for byte against the
64-bit oracle."""
import numpy as np
import pytest
import torch

from oracle import mx_oracle as mo
from paceserve_amd.kv_transfer import mx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_blocks_near_the_smallest_scale(gpu, dtype, fmt):
    rng = np.random.default_rng(17)
    N, P, H, D = 40, 16, 2, 64
    low = 24 if dtype is torch.float16 else 149 if dtype is torch.float32 else 133
    e = rng.integers(-low - 2, -100 if dtype is not torch.float16 else -8, (N, 2, P, H, D // 32, 1))
    x = rng.standard_normal((N, 2, P, H, D // 32, 32)) * 2.0 ** e.astype(np.float64)
    plain = [torch.from_numpy(x.reshape(N, 2, P, H, D)).to(dtype).to(gpu)]
    small = [mx.empty_cache(N, P, H, D, fmt, gpu)]
    ids = list(range(N))
    mx.quantize_pages(plain, ids, small, ids)
    values = plain[0].double().cpu().numpy()
    want = np.stack([np.concatenate([mo.page_half(values[i, h], fmt) for h in (0, 1)]) for i in range(N)])
    np.testing.assert_array_equal(small[0].cpu().numpy().reshape(N, -1), want)
    cache = torch.zeros_like(small[0])
    rows = plain[0].permute(0, 2, 1, 3, 4).reshape(N * P, 2 * H, D)
    i32 = dict(dtype=torch.int32, device=gpu)
    mx.append_paged_kv_cache_mx_indptr(rows[:, :H], rows[:, H:], torch.tensor([0, N * P], **i32), cache,
                                       torch.arange(N, **i32), torch.tensor([0, N], **i32), torch.tensor([P], **i32))
    assert torch.equal(cache, small[0])
    back = [torch.zeros_like(plain[0])]
    mx.dequantize_pages(small, ids, back, ids)
    data, byte = mo.split(small[0].cpu().numpy(), D)
    assert torch.equal(back[0].cpu(), torch.from_numpy(mo.values(data, byte, fmt)).to(dtype))
