"""rope and autograd on the GPU; test_gpu_rope.py holds its tolerances."""
import pytest
import torch
from torch.autograd import forward_ad

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


@pytest.mark.parametrize("dtype,dim,part,pairs", [(F32, 64, 64, False), (BF16, 128, 32, True), (BF16, 64, 34, False)])
@pytest.mark.parametrize("inverse", [False, True])
def test_a_tangent_is_rotated(cuda, dtype, dim, part, pairs, inverse):
    r = kvcache.Rotary(dim, theta=1e4, part=part, gain=1.2, interleaved=pairs)
    x, t = (torch.randn(2, 7, 3, dim, device="cuda").to(dtype) for _ in range(2))
    pos = torch.randint(0, 1000, (2, 7), dtype=torch.int32, device="cuda")
    off = torch.empty(1 + t.numel(), dtype=dtype, device="cuda")[1:].view(t.shape).copy_(t)
    for learns in (False, True):
        for tangent in (t, off):
            with forward_ad.dual_level():
                y = forward_ad.unpack_dual(kvcache.rope(forward_ad.make_dual(x.clone().requires_grad_(learns), tangent), r, pos, inverse))
                assert torch.equal(y.primal, kvcache.rope(x, r, pos, inverse)) and torch.equal(y.tangent, kvcache.rope(t, r, pos, inverse))


def test_what_is_saved_does_not_change_unnoticed(cuda):
    r, w, x = kvcache.Rotary(64, theta=1e4), torch.randn(2, 5, 3, 64, device="cuda", requires_grad=True), torch.randn(2, 5, 3, 64, device="cuda")
    y = (x * w).sum()
    kvcache.rope(x[:, 1:3], r, out=x[:, 1:3])
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.backward()
    with pytest.raises(ValueError, match="out"):
        kvcache.rope(x, r, out=w)
    with torch.inference_mode():
        z = torch.randn(2, 5, 3, 64, device="cuda")
        want = kvcache.rope(z, r)
        assert torch.equal(kvcache.rope(z, r, out=z), want)
