"""rope and autograd on the GPU; test_gpu_rope.py holds its tolerances."""
import pytest
import torch

from technograd_b200 import kvcache
from test_gpu_kvcache import BF16, F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("before", [1, 3, 8])
def test_a_gradient_that_begins_off_a_boundary(cuda, dtype, before):
    r = kvcache.Rotary(64, theta=1e4)
    x = torch.randn(2, 5, 3, 64, device="cuda").to(dtype).requires_grad_()
    w = torch.randn(before + x.numel(), device="cuda").to(dtype)
    (torch.cat([w[:before], kvcache.rope(x, r).flatten()]) * w).sum().backward()
    assert torch.equal(x.grad, kvcache.rope(w[before:].clone().view(x.shape), r, inverse=True))
