"""paged_attention has no backward pass, and says so (no GPU)."""
import pytest
import torch

from paceserve_amd.kv_transfer.attention import paged_attention


def test_tensors_that_require_gradients_are_refused():
    q, cache = torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 2, 16, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    for a, b in ((q.clone().requires_grad_(), cache), (q, cache.clone().requires_grad_())):
        with pytest.raises(ValueError, match="no backward"):
            paged_attention(a, b, i, i, i)
        for off in (torch.no_grad, torch.inference_mode):
            with off(), pytest.raises(ValueError, match="device tensor"):
                paged_attention(a, b, i, i, i)
