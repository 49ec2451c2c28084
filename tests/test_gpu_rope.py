"""Rotary positions and the append to the paged cache against the definition in 64 bits (GPU).

Tolerances, from the kernels' arithmetic (u = half a step of the output's type: 2^-24, 2^-11, 2^-8). cos and sin come from an
angle within 2^-24 of an eighth turn or less, through functions good to 2^-22, times the gain: each is off by at
most 2^-21 gain. y = x_a cos -+ x_b sin adds two roundings, so it is off by at most gain (|x_a| + |x_b|) (2^-21 + 2^-23) + u |y| (f16:
and 2^-25, half its least spacing). The norm's factor has at most 24 roundings of a sum, half of which the square root
leaves, three more and two products: 2^-24 (12 + 5) < 2^-19 of x."""
import math

import pytest
import torch

from technograd_b200 import _lib, kvcache
from test_gpu_kvcache import BF16, F16, F32, UNIT, Case, near, reported

pytestmark = pytest.mark.gpu


def turned(x, pos, freq, gain=1.0, pairs=False, inverse=False):
    """x f64 [b][t][heads][dim] rotated by pos [b][t], and the tolerance without the output's rounding."""
    half = len(freq)
    angle = pos.double()[:, :, None, None] * freq.cpu()
    c, s = gain * angle.cos(), gain * angle.sin() * (-1 if inverse else 1)
    y, tol = x.clone(), torch.zeros_like(x)
    a, b = (x[..., :half], x[..., half:2 * half]) if not pairs else (x[..., 0:2 * half:2], x[..., 1:2 * half:2])
    size = gain * (a.abs() + b.abs()) * (2.0 ** -21 + 2.0 ** -23)
    for i, z in enumerate((a * c - b * s, a * s + b * c)):
        where = (slice(i * half, i * half + half) if not pairs else slice(i, 2 * half, 2))
        y[..., where], tol[..., where] = z, size
    return y, tol


def normed(x, w, eps):
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double().cpu()


def close(got, want, tol, dtype, what="out"):
    near(got, want, tol + UNIT[dtype] * want.abs() + (2.0 ** -25 if dtype is F16 else 0), what)


def positions(B, T, seed, top=1 << 20):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-50, top, (B, T), generator=g, dtype=torch.int32)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim,part", [(8, 8), (64, 64), (80, 40), (80, 80), (128, 128), (128, 32), (128, 0), (136, 6), (256, 256), (256, 2), (72, 70)])
@pytest.mark.parametrize("pairs", [False, True])
def test_rope(cuda, dtype, dim, part, pairs):
    g = torch.Generator().manual_seed(1)
    for B, T, heads in ((1, 1, 1), (2, 5, 3), (3, 67, 17)):
        x = torch.randn(B, T, heads, dim, generator=g).to(dtype)
        r = kvcache.Rotary(dim, kvcache.rotary_frequencies(part, 1e6, 4.0, 32768).cuda(), gain=1.14, interleaved=pairs)
        pos = positions(B, T, 2)
        for inverse in (False, True):
            got = kvcache.rope(x.cuda(), r, pos.cuda(), inverse=inverse)
            want, tol = turned(x.double(), pos, r.freq, r.gain, pairs, inverse)
            close(got, want, tol, dtype)
        own = kvcache.rope(x.cuda(), r)  # positions 0, 1, ...
        want, tol = turned(x.double(), torch.arange(T).expand(B, T), r.freq, r.gain, pairs)
        close(own, want, tol, dtype)
        assert torch.equal(kvcache.rope(x.cuda(), r, torch.arange(T, dtype=torch.int32, device="cuda")), own)


def test_far_positions(cuda):
    """Positions to the ends of 32 bits, where an f32 angle would be off by hundreds of radians."""
    x = torch.randn(1, 6, 2, 128, generator=torch.Generator().manual_seed(3))
    pos = torch.tensor([[2 ** 31 - 1, -2 ** 31, 16777217, 2 ** 30 + 1, -1, 0]], dtype=torch.int32)
    r = kvcache.Rotary(128, theta=1e4)
    # the definition itself, in 64 bits, has angles within 2^-53 of theirs: 2^31 radians to 2^-22
    want, tol = turned(x.double(), pos, r.freq)
    size = x.abs()[..., :64] + x.abs()[..., 64:]
    tol += torch.cat([size, size], -1).double() * (pos.double().abs() * 2.0 ** -52)[:, :, None, None]
    close(kvcache.rope(x.cuda(), r, pos.cuda()), want, tol, F32)


def test_frequencies_of_any_size(cuda):
    """Of several turns a position, negative, zero; what is no number spoils its own pair only."""
    f = torch.tensor([20.0, -3.5, 0.0, 1e-300, math.pi, 1e6, math.nan, math.inf], dtype=torch.float64)
    x = torch.randn(1, 9, 1, 16, generator=torch.Generator().manual_seed(4))
    pos = torch.arange(9, dtype=torch.int32)[None]
    got = kvcache.rope(x.cuda(), kvcache.Rotary(16, f.cuda()), pos.cuda())
    want, tol = turned(x.double(), pos, torch.nan_to_num(f, 0, 0, 0))
    keep = [i for i in range(16) if i % 8 < 6]
    # (the product of a frequency in turns has 2^-53 of a number of up to 2^18 turns a position)
    close(got[..., keep], want[..., keep], tol[..., keep] + 2.0 ** -30, F32)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim,part", [(64, 6), (64, 32), (80, 20), (128, 34)])
@pytest.mark.parametrize("pairs", [False, True])
def test_what_passes_stays_as_it_is(cuda, dtype, dim, part, pairs):
    """Infinities and NaN behind the rotated part reach nothing, and are what they were."""
    x = torch.randn(2, 3, 5, dim, generator=torch.Generator().manual_seed(12)).to(dtype)
    r, pos = kvcache.Rotary(dim, theta=1e4, part=part, interleaved=pairs), positions(2, 3, 13)
    x[..., part:] = torch.tensor([math.inf, -math.inf, math.nan, -0.0]).to(dtype)[torch.arange(dim - part) % 4]
    got = kvcache.rope(x.cuda(), r, pos.cuda()).cpu()
    want, tol = turned(x[..., :part].double(), pos, r.freq, pairs=pairs)
    close(got[..., :part], want, tol, dtype)
    assert torch.equal(torch.nan_to_num(got[..., part:].float(), 7, 8, 9), torch.nan_to_num(x[..., part:].float(), 7, 8, 9))


@pytest.mark.parametrize("dtype,dim,part,pairs", [(BF16, 128, 128, False), (F16, 80, 20, False), (F32, 64, 64, True), (F16, 64, 48, True)])
def test_in_place_and_strided(cuda, dtype, dim, part, pairs):
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(3, 11, 9, dim, generator=g).to(dtype).cuda()
    r = kvcache.Rotary(dim, theta=1e4, part=part, interleaved=pairs)
    pos = positions(3, 11, 6).cuda()
    want = kvcache.rope(wide[:, :, 2:6].contiguous(), r, pos)
    before = wide.clone()
    assert torch.equal(kvcache.rope(wide[:, :, 2:6], r, pos), want) and torch.equal(wide, before)
    assert torch.equal(kvcache.rope(wide[:, :, 2:6].transpose(1, 2).contiguous().transpose(1, 2), r, pos), want)
    one = torch.randn(1, 1, 1, dim, generator=g).to(dtype).cuda()
    assert torch.equal(kvcache.rope(one.expand(3, 11, 4, dim), r, pos), kvcache.rope(one.expand(3, 11, 4, dim).contiguous(), r, pos))
    got = kvcache.rope(wide[:, :, 2:6], r, pos, out=wide[:, :, 2:6])
    before[:, :, 2:6] = want
    assert got.data_ptr() == wide[:, :, 2:6].data_ptr() and torch.equal(wide, before)
    back = kvcache.rope(want, r, pos, inverse=True).float()
    assert (back - kvcache.rope(kvcache.rope(back.to(dtype), r, pos), r, pos, inverse=True).float()).abs().max() <= 8 * UNIT[dtype] * back.abs().max()


@pytest.mark.parametrize("dim,part,pairs,inverse", [(64, 64, False, False), (64, 64, True, True), (32, 12, False, False)])
def test_gradient(cuda, dim, part, pairs, inverse):
    """Against the transposed rotation's formula, and against differences: a rotation is linear, so those of step 1 are the
    derivative but for roundings."""
    g = torch.Generator().manual_seed(7)
    B, T, H = 2, 5, 3
    x, w = (torch.randn(B, T, H, dim, generator=g) for _ in range(2))
    r = kvcache.Rotary(dim, theta=1e4, part=part, gain=1.2, interleaved=pairs)
    pos = positions(B, T, 8)
    leaf = x.cuda().requires_grad_()
    y = kvcache.rope(leaf, r, pos.cuda(), inverse=inverse)
    y.backward(w.cuda())
    want, tol = turned(w.double(), pos, r.freq, r.gain, pairs, not inverse)
    close(leaf.grad, want, tol, F32, "grad")
    for at in ((0, 0, 0, 0), (1, 4, 2, dim - 1), (1, 2, 1, part // 2), (0, 3, 2, part - 1)):
        up, down = x.clone(), x.clone()
        up[at] += 1
        down[at] -= 1
        two = [kvcache.rope(z.cuda(), r, pos.cuda(), inverse=inverse).double().cpu() for z in (up, down)]
        d = ((two[0] - two[1]) * w.double()).sum() / 2
        # the two rows' roundings: 2^-23 of elements of at most 1.2 * 2 * 5 in size, times the weights of the row's two elements
        assert abs(d - leaf.grad[at].cpu().double()) < 2.0 ** -20 * 12 * (1 + w[at[:3]].abs().max())


def test_gradients_of_odd_layout(cuda):
    """A gradient that arrives expanded or transposed, twice through the same graph, and of a gradient."""
    r = kvcache.Rotary(64, theta=1e4)
    x = torch.randn(2, 3, 4, 64, device="cuda", requires_grad=True)
    y = kvcache.rope(x, r)
    a, = torch.autograd.grad(y.sum(), x, retain_graph=True)
    b, = torch.autograd.grad(y, x, torch.ones(2, 3, 64, 4, device="cuda").transpose(2, 3), retain_graph=True)
    c, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(a, b) and torch.equal(a, c)
    w = torch.randn(2, 3, 4, 64, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(kvcache.rope(x, r), x, w, create_graph=True)
    h, = torch.autograd.grad(g, w, x.detach())
    assert torch.equal(h, kvcache.rope(x.detach(), r))


def test_rope_on_a_side_stream_and_in_a_graph(cuda):
    x, r, pos = torch.randn(5, 300, 8, 128, device="cuda").to(BF16), kvcache.Rotary(128, theta=1e6), positions(5, 300, 9).cuda()
    want = kvcache.rope(x, r, pos)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = kvcache.rope(x, r, pos)
    s.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = kvcache.rope(x, r, pos)
    pos += 3
    g.replay()
    assert torch.equal(got, kvcache.rope(x, r, pos)) and not torch.equal(got, want)


def test_forward_and_gradient_in_a_graph(cuda):
    r, x, w = kvcache.Rotary(64, theta=1e4), torch.randn(2, 9, 3, 64, device="cuda"), torch.randn(2, 9, 3, 64, device="cuda")
    leaf = x.clone().requires_grad_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(kvcache.rope(leaf, r), leaf, w)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = kvcache.rope(leaf, r)
        d, = torch.autograd.grad(y, leaf, w)
    with torch.no_grad():
        leaf += 1
    w *= 2
    g.replay()
    assert torch.equal(y, kvcache.rope(x + 1, r)) and torch.equal(d, kvcache.rope(w, r, inverse=True))


@pytest.mark.parametrize("part,pairs", [(128, False), (128, True), (100, False)])
def test_rope_past_32_bits(cuda, part, pairs):
    """Sequences 4 GB apart, in and out."""
    r = kvcache.Rotary(128, theta=1e6, part=part, interleaved=pairs)
    far = torch.empty(2, (1 << 31) + 4096, dtype=BF16, device="cuda")
    x = far[:, :3 * 2 * 128].view(2, 3, 2, 128)
    x.copy_(torch.randn(2, 3, 2, 128, generator=torch.Generator().manual_seed(14)))
    want = kvcache.rope(x.contiguous(), r)
    assert torch.equal(kvcache.rope(x, r), want) and torch.equal(kvcache.rope(x, r, out=x), want)


@pytest.mark.parametrize("tokens,heads,part", [(3000, 33, 64), (2500, 7, 64), (3000, 9, 20), (1, 1000, 64), (2100, 1, 64)])
@pytest.mark.parametrize("pairs", [False, True])
def test_many_tokens_and_heads(cuda, tokens, heads, part, pairs):
    """Both ways of sharing a token's rows among warps, with rows that do not fill one."""
    x = torch.randn(1, tokens, heads, 64, generator=torch.Generator().manual_seed(15))
    r, pos = kvcache.Rotary(64, theta=1e4, part=part, interleaved=pairs), positions(1, tokens, 16)
    want, tol = turned(x.double(), pos, r.freq, pairs=pairs)
    for dt in (BF16, F32):
        if dt is BF16:
            w, t = turned(x.to(BF16).double(), pos, r.freq, pairs=pairs)
        else:
            w, t = want, tol
        close(kvcache.rope(x.to(dt).cuda(), r, pos.cuda()), w, t, dt)


def test_rope_refusals(cuda):
    r, x = kvcache.Rotary(64, theta=1e4), torch.zeros(2, 3, 4, 64, device="cuda")
    pos = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for bad in (dict(x=x.double()), dict(x=x[0]), dict(x=x.transpose(2, 3)), dict(x=x.cpu()), dict(pos=pos.long()), dict(pos=pos[:1]), dict(pos=pos.cpu()),
                dict(x=x[..., :32]), dict(out=x.half()), dict(out=x[:1]), dict(out=x.view(2, 4, 3, 64).transpose(1, 2))):
        with pytest.raises(ValueError):
            kvcache.rope(**{**dict(x=x, rotary=r, pos=pos), **bad})
    odd = torch.zeros(2, 3, 4, 65, device="cuda")[..., 1:]
    for kw in (dict(x=odd), dict(x=x, pos=pos, out=torch.zeros(2, 3, 1, 64, device="cuda").expand(2, 3, 4, 64))):
        with pytest.raises(_lib.TgCudaError) as e:
            kvcache.rope(rotary=r, **kw)
        assert e.value.status == _lib.EINVAL
    for kw in (dict(freq=torch.ones(32, device="cuda")), dict(freq=torch.ones(33, dtype=torch.float64, device="cuda")), dict(part=63), dict(part=66),
               dict(freq=torch.ones(16, dtype=torch.float64, device="cuda"), part=30)):
        with pytest.raises(ValueError):
            kvcache.Rotary(64, **kw)
    with pytest.raises(ValueError):
        kvcache.rope(x.requires_grad_(), r, pos, out=torch.zeros_like(x))
    assert kvcache.rope(torch.zeros(0, 3, 4, 64, device="cuda"), r).shape == (0, 3, 4, 64)


# ---- append --------------------------------------------------------------------------------------------

def check_append(c, count=None, rotary=None, pos=None, q_norm=None, k_norm=None, keys=True, query=True, eps=1e-6):
    before = c.pk.clone(), c.pv.clone()
    dev = [None if x is None else x.cuda() for x in (pos, None if count is None else torch.tensor(count, dtype=torch.int32), q_norm, k_norm)]
    lens, q, k = kvcache.append(c.cache, c.kn.cuda(), c.vn.cuda(), q=c.q.cuda() if query else None, rotary=rotary, pos=dev[0], count=dev[1],
                                q_norm=dev[2], k_norm=dev[3], eps=eps, keys=keys)
    B, T = len(c.lens), c.T
    m = [T if count is None else max(0, min(T, n)) for n in count or [T] * B]
    assert lens.tolist() == [a + b for a, b in zip(c.lens, m)]
    at = pos if pos is not None else torch.tensor(c.lens)[:, None] + torch.arange(T)
    dead = torch.arange(T)[None] >= torch.tensor(m)[:, None]
    wants = []
    for x, w in ((c.q, q_norm), (c.kn, k_norm)):
        y, tol = x.double(), torch.zeros(1, dtype=torch.float64)
        if w is not None:
            y = normed(y, w, eps)
        if rotary is not None:
            slack = turned(y.abs() * 2.0 ** -19, at * 0, rotary.freq, rotary.gain, rotary.interleaved)[1] * 2.0 ** 21 if w is not None else 0  # gain (|x_a| + |x_b|) 2^-19
            y, tol = turned(y, at, rotary.freq, rotary.gain, rotary.interleaved)
            tol = tol + slack
        if w is not None:
            tol = tol + y.abs() * 2.0 ** -19
        wants.append((y.masked_fill(dead[..., None, None], 0), tol))
    if query:
        close(q, *wants[0], c.dtype, "q")
    if keys:
        close(k, *wants[1], c.dtype, "k")
    assert (q is None) == (not query) and (k is None) == (not keys)
    tol = wants[1][1].expand_as(wants[1][0])
    for b in range(B):
        p = torch.arange(c.lens[b], c.lens[b] + m[b])
        where = c.table[b].cpu()[p // c.page].long().cuda(), slice(None), (p % c.page).cuda()
        close(c.pk[where], wants[1][0][b, :m[b]], tol[b, :m[b]], c.dtype, "cached k")
        if keys:
            assert torch.equal(c.pk[where], k[b, :m[b]])
        assert torch.equal(c.pv[where].cpu(), c.vn[b, :m[b]])
        before[0][where], before[1][where] = c.pk[where], c.pv[where]
    for x, y in zip((c.pk, c.pv), before):  # nothing else is written
        assert torch.equal(torch.nan_to_num(x.float(), 777), torch.nan_to_num(y.float(), 777))
    return lens, q, k


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim,part,page,order,tokens,nkv,group", [(8, 4, 5, "head", 1, 2, 2), (128, 128, 16, "pos", 9, 8, 2), (80, 20, 3, "head", 64, 1, 3),
                                                                  (256, 256, 64, "pos", 130, 2, 1), (64, 64, 24, "pos", 1, 1, 1), (136, 130, 16, "head", 33, 3, 5)])
@pytest.mark.parametrize("pairs", [False, True])
def test_append(cuda, dtype, dim, part, page, order, tokens, nkv, group, pairs):
    g = torch.Generator().manual_seed(10)
    w = [1 + 0.3 * torch.randn(dim, generator=g) for _ in range(2)]
    r = kvcache.Rotary(dim, theta=1e6, part=part, gain=1.1, interleaved=pairs)
    for kw in (dict(rotary=r, q_norm=w[0], k_norm=w[1]), dict(rotary=r, pos=positions(4, tokens, 11), keys=False), dict(), dict(rotary=r, k_norm=w[1], query=False),
               dict(q_norm=w[0])):
        c = Case([0, 33, 64, 7], nkv, group, dim, page, order, dtype, tokens, room=tokens)
        check_append(c, [tokens, tokens // 2, 0, min(1, tokens)], **kw)
    check_append(Case([40], nkv, group, dim, page, order, dtype, tokens, room=tokens), rotary=r)


def test_append_counts_out_of_range(cuda):
    c = Case([5, 6, 7], 2, 2, 64, 16, "head", BF16, 4, room=4)
    check_append(c, [9, -3, 4], kvcache.Rotary(64, theta=1e4))


def test_append_of_a_projection(cuda):
    """q, k and v as views of one projection's rows, in place and on a side stream, and in a graph."""
    c = Case([100, 37, 0], 2, 4, 64, 16, "pos", BF16, 6, room=12)
    x = torch.empty(3, 6, 12, 64, dtype=BF16, device="cuda")
    q, k, v = x.split([8, 2, 2], 2)
    q.copy_(c.q), k.copy_(c.kn), v.copy_(c.vn)
    r = kvcache.Rotary(64, theta=1e4)
    want = kvcache.append(c.cache, c.kn.cuda(), c.vn.cuda(), q=c.q.cuda(), rotary=r, keys=True)
    pools = c.pk.clone(), c.pv.clone()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = kvcache.append(c.cache, k, v, q=q, rotary=r, keys=True)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = kvcache.append(c.cache, k, v, q=q, rotary=r, keys=True)
    c.pk.zero_(), c.pv.zero_()
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for b, n in enumerate(c.lens):
        p = torch.arange(n, n + 6)
        where = c.table[b].cpu()[p // 16].long().cuda(), slice(None), (p % 16).cuda()
        assert torch.equal(c.pk[where], pools[0][where]) and torch.equal(c.pv[where], pools[1][where])
    d = kvcache._drafts(c.cache, q, k, v, None, None, 1.0)  # q and k themselves as q_out and k_out
    lens, e = torch.empty_like(c.len), (*q.stride()[:3],)
    _lib.check(cuda.tg_cuda_kv_append(c.cache._at, d, r._pack(None, 3, 6, 0, 64), None, None, 1e-6, q.data_ptr(), *e, k.data_ptr(), *e, lens.data_ptr(),
                                      torch.cuda.current_stream().cuda_stream))
    assert torch.equal(q, want[1]) and torch.equal(k, want[2]) and torch.equal(v.cpu(), c.vn)


def test_append_past_32_bits(cuda):
    c = Case([130], 1, 2, 128, 64, "head", BF16, 3, room=3)
    pages = (1 << 32) // (64 * 128 * 2) + 40
    pk, pv = (torch.zeros(pages, 1, 64, 128, dtype=BF16, device="cuda") for _ in range(2))
    where = torch.tensor([[1, 2, pages - 7, 3]], dtype=torch.int32, device="cuda")
    cache = kvcache.PagedKV(pk, pv, where, c.len, max_len=130)
    _, _, k = kvcache.append(cache, c.kn.cuda(), c.vn.cuda(), rotary=kvcache.Rotary(128, theta=1e6), keys=True)
    assert torch.equal(pk[pages - 7, 0, 2:5], k[0, :, 0]) and torch.equal(pv[pages - 7, 0, 2:5].cpu(), c.vn[0, :, 0])
    assert pk.count_nonzero() == k.count_nonzero() and not pk[:, :, :2].any()


def test_append_device_data_out_of_range_is_reported(cuda):
    c = Case([40, 20], 2, 2, 64, 16, "head", BF16, 3, room=3)
    k, v = c.kn.cuda(), c.vn.cuda()
    good = lambda: kvcache.tree_attention(c.cache, c.q.cuda(), k, v)  # noqa: E731
    pools = c.pk.clone(), c.pv.clone()
    t = c.table.clone()
    t[:, 1:] = 10 ** 6
    kvcache.append(kvcache.PagedKV(c.pk, c.pv, t, c.len, max_len=40), k, v)
    assert "page number" in reported(good)
    room = kvcache.PagedKV(c.pk, c.pv, c.table[:, :2].contiguous(), torch.tensor([32, 32], dtype=torch.int32, device="cuda"), max_len=32)
    kvcache.append(room, k, v, rotary=kvcache.Rotary(64, theta=1e4))
    assert "past the table" in reported(good)
    for x, y in zip((c.pk, c.pv), pools):
        assert torch.equal(torch.nan_to_num(x.float(), 777), torch.nan_to_num(y.float(), 777))
    kvcache.append(c.cache.with_lens(torch.tensor([41, -1], dtype=torch.int32, device="cuda"), 40), k, v)
    assert "len" in reported(good)
