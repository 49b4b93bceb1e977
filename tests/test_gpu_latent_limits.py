"""paged_latent_attention and latent_prompt_attention (HIP) at the ends of their ranges,
against 64 bits."""
import math

import numpy as np
import pytest
import torch

from paceserve_amd.kv_transfer import latent

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


def check_one_above(out, lse, scores, values, dtype):
    """Rows out [..., D] that all see tokens of `scores` (natural units) and `values` [n, D].
    The largest weight is 1, which no type rounds: what the others' rounding moves is half a
    step of what they add (and the sum over all is float32's)."""
    s, v, eps = np.asarray(scores), values.astype(np.float64), torch.finfo(dtype).eps
    p = np.exp(s - s.max())
    want, rest = p @ v / p.sum(), np.delete(p, s.argmax()) @ np.abs(np.delete(v, s.argmax(), 0)) / p.sum()
    # scores of at most 2^5 are off by 2^-19 at most (2^-24 of them in float32, and the scale),
    # weights by as much and by the exponential's 2^-21
    f32 = 2.0 ** -17 * (p @ np.abs(v)) / p.sum()
    bound = eps / 2 * (np.abs(want) + rest) * (1 + eps) + f32 + (2.0 ** -25 if dtype is FP16 else 0.0)
    off = np.abs(out.double().cpu().numpy() - want) / bound
    assert off.max() <= 1, f"off by {off.max():.3g} of its bound"
    total = s.max() + math.log(p.sum())
    assert np.abs(lse.double().cpu().numpy() - total).max() <= 2.0 ** -17 * (1 + abs(total))


@pytest.mark.parametrize("above", [0.12, 1.0037, 2.08298, 2.7, 3.0])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,L", [(1, 512), (16, 256), (32, 512), (20, 256), (128, 512), (40, 256)])
def test_a_token_above_those_before_it_counts_in_full(gpu, heads, L, dtype, above):
    """A first token, many of next to no weight, then one some way above the first: its weight is
    the unit, whatever the maximum was before.  (2.08298 is log 8.0283, nearly midway between
    two of bfloat16's numbers.)  All on one page, which is never cut."""
    rng = np.random.default_rng(heads)
    n, P, at, batch = 100, 128, 70, 3
    rank = np.full(n, -8.0)
    rank[0], rank[at] = 0.0, 1.0
    x = torch.zeros((n, L + 64), dtype=torch.float64)
    x[:, :L] = torch.from_numpy(rng.standard_normal((n, L)))
    x[:, L] = torch.from_numpy(rank)
    x = x.to(dtype)
    cache = latent.empty_cache(1, P, L, dtype, gpu)
    cache.view(-1, L + 64)[:n] = x.to(gpu)
    q = torch.zeros((batch, heads, L + 64), dtype=dtype, device=gpu)
    q[..., L] = 1.0
    out, lse = latent.paged_latent_attention(q, cache, i32([0] * batch, gpu), i32(np.arange(batch + 1), gpu),
                                             i32([n] * batch, gpu), sm_scale=above, return_lse=True)
    torch.cuda.synchronize()
    assert torch.equal(out, out[:1, :1].expand_as(out)) and torch.equal(lse, lse[:1, :1].expand_as(lse))
    check_one_above(out[:2], lse[:2], rank * above, x[:, :L].double().numpy(), dtype)


@pytest.mark.parametrize("above", [0.12, 1.0037, 2.08298, 2.7, 3.0])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
def test_a_key_above_those_before_it_counts_in_full(gpu, D, dtype, above):
    rng = np.random.default_rng(D)
    n, t, at, heads = 300, 150, 70, 500
    assert latent._prompt_workspace_bytes(t, n, 1, heads, D, 0) == 0          # no keys are dealt out
    rank = np.full(n, -8.0)
    rank[0], rank[at] = 0.0, 1.0
    value = torch.from_numpy(rng.standard_normal((n, 1, D))).to(dtype)
    rope = torch.zeros((n, 64), dtype=dtype, device=gpu)
    rope[:, 3] = torch.from_numpy(rank)
    q = torch.zeros((t, heads, D + 64), dtype=dtype, device=gpu)
    q[..., D + 3] = 1.0
    key = torch.zeros((n, 1, D), dtype=dtype, device=gpu)
    out, lse = latent.latent_prompt_attention(q, key.expand(-1, heads, -1), rope, value.to(gpu).expand(-1, heads, -1),
                                              i32([0, t], gpu), i32([0, n], gpu), sm_scale=above, causal=False,
                                              return_lse=True)
    torch.cuda.synchronize()
    assert torch.equal(out, out[:1, :1].expand_as(out)) and torch.equal(lse, lse[:1, :1].expand_as(lse))
    check_one_above(out[:, 0], lse[:, 0], rank * above, value[:, 0].double().numpy(), dtype)
