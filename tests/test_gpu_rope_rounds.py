"""Rotations of many tokens against the same tokens a few at a time (GPU): how a warp takes its rows changes no bit."""
import pytest
import torch

from technograd_b200 import kvcache
from test_gpu_kvcache import BF16, F16, F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim,heads,tokens", [(BF16, 128, 16, 7001), (BF16, 128, 17, 6001), (F16, 80, 32, 3500), (F32, 128, 8, 12400), (F32, 68, 15, 7001), (BF16, 256, 8, 12300),
                                                    (F16, 8, 128, 800), (BF16, 64, 1, 100001)])
@pytest.mark.parametrize("pairs", [False, True])
def test_rope(cuda, dtype, dim, heads, tokens, pairs):
    x = torch.randn(1, tokens, heads, dim, device="cuda").to(dtype)
    r = kvcache.Rotary(dim, theta=1e5, part=dim // 16 * 16 or dim, interleaved=pairs)
    pos = torch.randint(0, 1 << 20, (tokens,), dtype=torch.int32, device="cuda")
    got = kvcache.rope(x, r, pos)
    for at in range(0, tokens, 700):
        assert torch.equal(got[:, at:at + 700], kvcache.rope(x[:, at:at + 700], r, pos[at:at + 700]))
    assert torch.equal(kvcache.rope(x, r, pos, out=x), got) and got.data_ptr() != x.data_ptr()


@pytest.mark.parametrize("dtype,dim,nq,nkv", [(BF16, 128, 16, 8), (F16, 128, 32, 8), (BF16, 128, 33, 11), (F32, 80, 16, 8), (BF16, 128, 8, 1)])
@pytest.mark.parametrize("norm", [False, True])
def test_append(cuda, dtype, dim, nq, nkv, norm):
    B, T, page = 3, 2100, 16
    cols = -(-T // page)
    x = torch.randn(B, T, nq + 2 * nkv, dim, device="cuda").to(dtype)
    q, k, v = x.split([nq, nkv, nkv], 2)
    r, table = kvcache.Rotary(dim, theta=1e5), torch.randperm(B * cols, device="cuda").int().view(B, cols)
    kw = dict(rotary=r, keys=True)
    if norm:
        kw.update(q_norm=1 + torch.randn(dim, device="cuda") / 8, k_norm=1 + torch.randn(dim, device="cuda") / 8)

    def pools():
        return tuple(torch.zeros(B * cols, nkv, page, dim, dtype=dtype, device="cuda") for _ in range(2))
    once, parts = pools(), pools()
    none = torch.zeros(B, dtype=torch.int32, device="cuda")
    lens, qr, kr = kvcache.append(kvcache.PagedKV(*once, table, none, max_len=0), k, v, q=q, **kw)
    assert lens.tolist() == [T] * B
    at = none
    for i in range(0, T, 300):
        now = slice(i, i + 300)
        at, a, b = kvcache.append(kvcache.PagedKV(*parts, table, at, max_len=i), k[:, now], v[:, now], q=q[:, now], **kw)
        assert torch.equal(a, qr[:, now]) and torch.equal(b, kr[:, now])
    assert torch.equal(once[0], parts[0]) and torch.equal(once[1], parts[1])
