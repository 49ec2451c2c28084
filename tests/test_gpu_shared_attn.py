"""Attention below shared prefixes against the definition in 64 bits (GPU): cases, definition and tolerances of
test_gpu_kvcache.py (the join's factors are four roundings of 2^-22, far within its 2^-18), and half of f16's least spacing more."""
import math

import pytest
import torch

from technograd_b200 import _lib, kvcache
from test_gpu_kvcache import BF16, F16, F32, INF, Case, attend, bits, near, plain, random_mask, reported

pytestmark = pytest.mark.gpu


class Shared(Case):
    """A Case whose groups' first positions lie in the same pages. groups: (first, members, pages, positions said to be shared);
    own: positions of every sequence behind its group's pages."""

    def __init__(self, own, groups, nkv=2, group=2, dim=128, page=16, order="head", dtype=BF16, tokens=1, seed=1, room=0, max_own=None):
        lens = list(own)
        for first, members, pages, _ in groups:
            for b in range(first, first + members):
                lens[b] += pages * page
        super().__init__(lens, nkv, group, dim, page, order, dtype, tokens, seed, room=room)
        table = self.table.cpu()
        for first, members, pages, _ in groups:
            for b in range(first + 1, first + members):
                gone = table[b, :pages].long()  # theirs are nobody's now
                self.pk[gone.cuda()], self.pv[gone.cuda()] = math.nan, math.nan
                table[b, :pages] = table[first, :pages]
                self.k[b][:pages * page], self.v[b][:pages * page] = self.k[first][:pages * page], self.v[first][:pages * page]
        self.table = table.cuda()
        self.cache = kvcache.PagedKV(self.pk, self.pv, self.table, self.len, max_len=max(lens))
        self.prefix = kvcache.SharedPrefix(self.cache, [(f, m, s) for f, m, _, s in groups], max_own=max(own) if max_own is None else max_own, always=True)


def run(c, mask=None, count=None, **kw):
    dev = dict(mask=None if mask is None else mask.cuda(), count=None if count is None else torch.tensor(count, dtype=torch.int32, device="cuda"))
    return kvcache.shared_attention(c.cache, c.prefix, c.q.cuda(), c.kn.cuda(), c.vn.cuda(), **dev, **kw)


def check(c, mask=None, count=None):
    got, want = run(c, mask, count), plain(c, mask, count)
    near(got[0], want[0], want[2] + (2.0 ** -25 if c.dtype is F16 else 0), "out")
    near(got[1], want[1], want[3], "lse")
    return got


GROUPS = [(1, 3, 5, 80), (4, 2, 9, 144), (7, 1, 2, 32)]
OWN = [70, 0, 1, 259, 30, 31, 0, 128, 77]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [8, 64, 80, 128, 136, 256])
@pytest.mark.parametrize("tokens,nkv,group", [(1, 2, 2), (7, 1, 3), (33, 2, 1), (64, 1, 4)])
def test_shapes(cuda, dtype, dim, tokens, nkv, group):
    c = Shared(OWN, GROUPS, nkv, group, dim, 16, "head", dtype, tokens)
    check(c, random_mask(9, tokens, 3), [tokens, tokens, (tokens + 1) // 2, 0, tokens, 1, tokens, tokens, 0])


@pytest.mark.parametrize("page,order", [(1, "pos"), (3, "head"), (5, "pos"), (8, "head"), (16, "pos"), (24, "head"), (32, "pos"), (64, "head"), (128, "pos"), (192, "head"), (1000, "pos")])
@pytest.mark.parametrize("dtype,tokens", [(F32, 1), (F32, 12), (BF16, 1), (F16, 40)])
def test_pages(cuda, page, order, dtype, tokens):
    n = -(-300 // page)
    c = Shared([15, 16, 1, 63, 300], [(0, 4, n, n * page)], 2, 2, 128, page, order, dtype, tokens)
    check(c, random_mask(5, tokens, 4))


@pytest.mark.parametrize("shared", [0, 1, 15, 16, 63, 64, 65, 127, 128, 129, 200, 255])
@pytest.mark.parametrize("dtype,tokens,page", [(F32, 2, 16), (BF16, 1, 16), (BF16, 24, 64), (F16, 3, 128), (BF16, 1, 256)])
def test_less_is_shared_than_could_be(cuda, shared, dtype, tokens, page):
    """A prefix that ends anywhere, within a page, a tile and a box."""
    check(Shared([40, 3, 0, 90], [(0, 3, 256 // page, shared)], 2, 2, 64, page, "pos", dtype, tokens))


@pytest.mark.parametrize("dtype,tokens,members,pages", [(BF16, 1, 1, 1200), (F16, 5, 2, 700), (F32, 1, 3, 900), (BF16, 13, 40, 70), (F32, 9, 11, 60), (BF16, 64, 5, 130)])
def test_long_prefixes_and_many_rows(cuda, dtype, tokens, members, pages):
    """Prefixes over many CTAs, groups of many row tiles."""
    own = [(b * 37) % 90 for b in range(members + 1)]
    check(Shared(own, [(0, members, pages, pages * 16)], 2, 4, 128, 16, "head", dtype, tokens), random_mask(members + 1, tokens, 5))


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F32, 64), (F16, 256)])
def test_many_groups(cuda, dtype, dim):
    """More groups than threads look through them at once, some of one sequence, some that share nothing; sequences in none between them."""
    groups, at, own = [], 0, []
    for i in range(260):
        members, pages = 1 + i % 3, i % 5
        groups.append((at, members, pages, pages * 16))
        at += members + (i % 7 == 0)
    own = [(b * 11) % 40 for b in range(at)]
    check(Shared(own, groups, 1, 2, dim, 16, "head", dtype, 2))


@pytest.mark.parametrize("dim", [4, 64, 68, 128, 256])
@pytest.mark.parametrize("members,tokens,group", [(1, 1, 1), (2, 1, 2), (2, 2, 2), (3, 1, 3), (4, 1, 2), (2, 4, 1), (8, 1, 1), (9, 1, 1)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_few_rows_in_all(cuda, dtype, dim, members, tokens, group):
    """1 to 9 rows a key head of all sequences together: f32 takes the FMA units up to 8."""
    if dtype is BF16 and dim % 8:
        return
    for pages in (1, 9, 130):
        check(Shared([7, 0, 40, 1, 2, 3, 90, 5, 6][:members], [(0, members, pages, pages * 16)], 2, group, dim, 16, "pos", dtype, tokens))


@pytest.mark.parametrize("max_own", [0, 1, 10 ** 6])
@pytest.mark.parametrize("dtype,tokens", [(F32, 1), (BF16, 1), (BF16, 30)])
def test_max_own_is_a_hint(cuda, max_own, dtype, tokens):
    check(Shared([900, 5, 0, 1300], [(0, 3, 20, 320)], 2, 2, 128, 16, "head", dtype, tokens, max_own=max_own))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens", [4, 40])
def test_masked_rows_may_hold_anything(cuda, dtype, tokens):
    c = Shared([21, 0, 400], [(0, 2, 6, 96)], 2, 2, 128, 16, "head", dtype, tokens)
    mask = random_mask(3, tokens, 8) & ~((1 << 1) | (1 << (tokens - 1)))
    for x, y in ((c.kn, math.nan), (c.vn, INF)):
        x[:, 1] = y
        x[:, tokens - 1] = -INF if y == INF else y
    check(c, mask, [tokens, tokens, tokens - 1])
    seen = mask.clone()
    seen[:, 0] |= 2
    out, lse = run(c, seen, [tokens, tokens, tokens - 1])
    want = plain(c, mask, [tokens, tokens, tokens - 1])
    assert torch.isnan(out[:, 0].float()).all() and torch.isnan(lse[:, 0]).all()
    near(out[:, 1:], want[0][:, 1:], want[2][:, 1:] + 2.0 ** -25, "out")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_all_keys_of_one_part_weigh_nothing(cuda, dtype):
    """Scores thousands apart between the prefix and what follows it; nothing seen but the prefix, and only infinitely low scores."""
    c = Shared([500, 80, 1], [(0, 3, 10, 160)], 2, 2, 64, 16, "head", dtype, 3)
    c.q *= 60
    check(c)
    c.q *= 0
    check(c)
    c = Shared([0, 0], [(0, 2, 10, 160)], 2, 2, 64, 16, "head", dtype, 3)
    check(c, torch.zeros(2, 3, dtype=torch.int64))
    c.pk[:] = -INF  # a score of -infinity in every cached place
    c.q = c.q.abs() + 0.5
    out, lse = run(c, torch.zeros(2, 3, dtype=torch.int64))
    assert not out.any() and (lse == -INF).all()
    c.kn[:] = 0
    out, lse = run(c, bits([[1, 2, 4]] * 2))  # each sees itself alone
    near(out, c.vn.repeat_interleave(2, 2).double(), torch.zeros_like(out, dtype=torch.float64).cpu() + 2.0 ** -20, "out")


def test_same_as_without_sharing(cuda):
    """The attention of each sequence by itself, and of a batch that shares nothing, which is the same kernel's."""
    c = Shared(OWN, GROUPS, 2, 2, 128, 16, "head", BF16, 5)
    got, want = run(c), attend(c)
    # both are within an f32 softmax of the definition and then rounded once: apart by one step at most
    assert (got[0].float() - want[0].float()).abs().max() <= 2.0 ** -7 * want[0].float().abs().max() and (got[1] - want[1]).abs().max() < 1e-4
    c.prefix = kvcache.SharedPrefix(c.cache, [])
    none = run(c)
    assert torch.equal(none[0], want[0]) and torch.equal(none[1], want[1])
    c.prefix = kvcache.SharedPrefix(c.cache, [(0, 9, 0)], always=True)
    none = run(c)
    assert torch.equal(none[0], want[0]) and torch.equal(none[1], want[1])
    c.prefix = kvcache.SharedPrefix(c.cache, [(f, m, s) for f, m, _, s in GROUPS])  # so small that sharing costs more
    none = run(c)
    assert torch.equal(none[0], want[0]) and torch.equal(none[1], want[1])


@pytest.mark.parametrize("dtype,seqs,pages", [(BF16, 40, 130), (F32, 24, 200), (F16, 8, 300)])
def test_where_sharing_pays(cuda, dtype, seqs, pages):
    """Without being told to, and with the same bits as when told."""
    c = Shared([b % 50 for b in range(seqs)], [(0, seqs, pages, pages * 16)], 8, 2, 128, 16, "head", dtype, 1)
    want = check(c)
    c.prefix = kvcache.SharedPrefix(c.cache, [(0, seqs, pages * 16)], max_own=49)
    got = run(c)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_strides_and_scale(cuda):
    c = Shared([100, 37, 9], [(0, 2, 8, 128)], 2, 4, 64, 16, "head", BF16, 6)
    B, T, nq, D = c.q.shape
    x = torch.empty(B, T, nq + 2 * c.nkv, D, dtype=BF16, device="cuda")
    q, k, v = x.split([nq, c.nkv, c.nkv], 2)
    q.copy_(c.q), k.copy_(c.kn), v.copy_(c.vn)
    got = kvcache.shared_attention(c.cache, c.prefix, q, k, v, scale=0.3)
    want = plain(c, scale=0.3)
    near(got[0], want[0], want[2], "out")
    near(got[1], want[1], want[3], "lse")
    turned = [y.transpose(1, 2).contiguous().transpose(1, 2) for y in (q, k, v)]
    again = kvcache.shared_attention(c.cache, c.prefix, *turned, scale=0.3)
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])
    for scale in (-0.2, 0.0):
        flip = Shared([100, 37, 9], [(0, 2, 8, 128)], 2, 4, 64, 16, "head", BF16, 6)
        flip.q = -flip.q if scale < 0 else flip.q * 0
        got, want = run(c, scale=scale), plain(flip, scale=abs(scale) or 0.1)
        near(got[0], want[0], want[2], "out")
        near(got[1], want[1], want[3], "lse")


def test_again_on_side_streams_and_back_to_back(cuda):
    """Many calls in a row, whose kernels overlap, and on two streams at once: the same bits every time."""
    cs = [Shared([b * 9 for b in range(m)], [(0, m, 90, 1440)], 2, 2, 128, 16, "head", dt, t, seed=s) for s, (dt, t, m) in enumerate([(BF16, 1, 30), (F32, 2, 7), (F16, 40, 9)])]
    args = [(c.cache, c.prefix, c.q.cuda(), c.kn.cuda(), c.vn.cuda()) for c in cs]
    want = [kvcache.shared_attention(*a) for a in args]
    torch.cuda.synchronize()
    s1, s2, got = torch.cuda.Stream(), torch.cuda.Stream(), []
    for i in range(30):
        with torch.cuda.stream((s1, s2)[i % 2]):
            got.append([kvcache.shared_attention(*a) for a in args])
    torch.cuda.synchronize()
    for g in got:
        for x, y in zip(g, want):
            assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


def test_in_a_graph_with_changing_lengths(cuda):
    c = Shared([40, 30, 7], [(0, 2, 20, 320)], 2, 2, 128, 16, "head", BF16, 2)
    q, k, v = c.q.cuda(), c.kn.cuda(), c.vn.cuda()
    kvcache.shared_attention(c.cache, c.prefix, q, k, v)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = kvcache.shared_attention(c.cache, c.prefix, q, k, v)
    for cut in (0, 5, 20):
        c.len -= torch.tensor([cut, cut, min(cut, 3)], dtype=torch.int32, device="cuda")
        g.replay()
        want = kvcache.shared_attention(c.cache, c.prefix, q, k, v)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_offsets_past_32_bits(cuda):
    """A pool of more than 2^32 bytes whose used pages lie at its end, and queries as far apart."""
    c = Shared([70, 40], [(0, 2, 2, 128)], 1, 2, 128, 64, "head", BF16, 3)
    pages = (1 << 32) // (64 * 128 * 2) + 40
    pk, pv = (torch.zeros(pages, 1, 64, 128, dtype=BF16, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, pages - 30, pages - 7, pages - 3], [pages - 1, pages - 30, pages - 2, 0]], dtype=torch.int32, device="cuda")
    for b in range(2):
        for i in range(-(-c.lens[b] // 64)):
            pk[table[b, i]], pv[table[b, i]] = c.pk[c.table[b, i]], c.pv[c.table[b, i]]
    c.cache = kvcache.PagedKV(pk, pv, table, c.len, max_len=max(c.lens))
    check(c)
    far = torch.empty(2, (1 << 31) + 4096, dtype=BF16, device="cuda")  # q's sequences 4 GB apart
    q = far[:, :3 * 2 * 128].view(2, 3, 2, 128)
    q.copy_(c.q)
    got, want = kvcache.shared_attention(c.cache, c.prefix, q, c.kn.cuda(), c.vn.cuda()), plain(c)
    near(got[0], want[0], want[2], "out")


def test_device_data_that_does_not_suit_is_reported(cuda):
    """Lists that overlap, lengths below the prefix, numbers out of range: the call ends, stays in bounds, and a later one says so."""
    c = Shared([40, 20, 10, 30], [(0, 2, 4, 64), (2, 2, 3, 48)], 2, 2, 64, 16, "head", BF16, 3)
    q, k, v = c.q.cuda(), c.kn.cuda(), c.vn.cuda()
    good = lambda: kvcache.shared_attention(c.cache, c.prefix, q, k, v)  # noqa: E731
    good()
    fields = dict(first=0, members=2, shared=4, group=6)
    for name, values in (("shared", [65, 48]), ("shared", [-5, 48]), ("shared", [2 ** 31 - 1, -2 ** 31]), ("first", [0, 1]), ("first", [-1, 2]), ("first", [10 ** 6, 2]),
                         ("members", [2, 3]), ("members", [2 ** 31 - 1, 2]), ("members", [-7, 2]), ("members", [1, 2]), ("group", [0, 0, 2, 1]), ("group", [-2, 0, 1, 1]),
                         ("group", [1, 0, 0, 1])):
        x = kvcache.SharedPrefix(c.cache, [(0, 2, 64), (2, 2, 48)], always=True)
        x._held[fields[name]:fields[name] + len(values)] = torch.tensor(values, dtype=torch.int32, device="cuda")
        kvcache.shared_attention(c.cache, x, q, k, v)
        assert "group of sequences" in reported(good), (name, values)
    n = torch.tensor([104, 60, 58, 78], dtype=torch.int32, device="cuda")  # the second has less than its group shares
    kvcache.shared_attention(c.cache.with_lens(n, 104), c.prefix, q, k, v)
    assert "group of sequences" in reported(good)
    t = c.table.clone()
    t[0, 1] = 10 ** 6
    out, _ = kvcache.shared_attention(kvcache.PagedKV(c.pk, c.pv, t, c.len, max_len=104), c.prefix, q, k, v)
    assert torch.isfinite(out.float()).all() and "page number" in reported(good)


def test_refusals(cuda):
    c = Shared([40, 20], [(0, 2, 4, 64)], 2, 2, 64, 16, "head", BF16, 3)
    q, k, v = c.q.cuda(), c.kn.cuda(), c.vn.cuda()
    wide = torch.zeros(2, 65, 4, 64, dtype=BF16, device="cuda")
    with pytest.raises(_lib.TgCudaError) as e:
        kvcache.shared_attention(c.cache, c.prefix, wide, wide[:, :, :2], wide[:, :, :2])
    assert e.value.status == _lib.EINVAL
    other = Shared([40, 20, 1], [(0, 2, 4, 64)], 2, 2, 64, 16, "head", BF16, 3)
    with pytest.raises(ValueError):
        kvcache.shared_attention(c.cache, other.prefix, q, k, v)
    with pytest.raises(ValueError):
        kvcache.shared_attention(c.cache.with_lens(c.len, 63), c.prefix, q, k, v)
    d = kvcache._drafts(c.cache, q, k, v, None, None, None)
    n = cuda.tg_cuda_shared_attn_workspace(c.cache._at, d, c.prefix._at)
    out, lse, work = torch.empty_like(q), torch.empty(2, 3, 4, device="cuda"), torch.empty(n, dtype=torch.uint8, device="cuda")
    for w, size in ((None, n), (work.data_ptr(), n - 1), (work.data_ptr() + 8, n)):
        assert cuda.tg_cuda_shared_attn(c.cache._at, d, c.prefix._at, out.data_ptr(), *out.stride()[:3], lse.data_ptr(), w, size, None) == _lib.EINVAL


def test_a_decode_step_together(cuda):
    """Prompts of which the first half is common, then decode steps of one token: append with norm and rotation, attention below the shared prefix, as a server
    runs them, against the definition in 64 bits of the whole."""
    B, T, nq, nkv, dim, page, half = 5, 96, 4, 2, 64, 16, 48
    g = torch.Generator().manual_seed(20)
    x = torch.randn(B, T + 3, nq + 2 * nkv, dim, generator=g)
    x[1:, :half] = x[:1, :half]  # the common half
    x = x.to(BF16)
    w = [1 + 0.2 * torch.randn(dim, generator=g) for _ in range(2)]
    cols = -(-(T + 3) // page)
    table = torch.randperm(B * cols, generator=g).int().view(B, cols)
    table[1:, :half // page] = table[0, :half // page]
    pools = [torch.full((B * cols, nkv, page, dim), math.nan, dtype=BF16, device="cuda") for _ in range(2)]
    rotary = kvcache.Rotary(dim, theta=1e6)
    norms = dict(q_norm=w[0].cuda(), k_norm=w[1].cuda())
    dx = x.cuda()
    q, k, v = dx.split([nq, nkv, nkv], 2)

    # the common half once, then each sequence's own part of the prompt
    one = kvcache.PagedKV(*pools, table[:1].cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"), max_len=0)
    lens, _, _ = kvcache.append(one, k[:1, :half], v[:1, :half], rotary=rotary, k_norm=norms["k_norm"])
    assert lens.tolist() == [half]
    cache = kvcache.PagedKV(*pools, table.cuda(), lens.expand(B).contiguous(), max_len=half)
    prefix = kvcache.SharedPrefix(cache, [(0, B, half)], max_own=T + 3 - half, always=True)
    lens, _, _ = kvcache.append(cache, k[:, half:T], v[:, half:T], rotary=rotary, k_norm=norms["k_norm"])
    outs = []
    for t in range(T, T + 3):
        cache = cache.with_lens(lens, t)
        now = slice(t, t + 1)
        lens, qr, kr = kvcache.append(cache, k[:, now], v[:, now], q=q[:, now], rotary=rotary, keys=True, **norms)
        outs.append(kvcache.shared_attention(cache, prefix, qr, kr, v[:, now])[0])
    assert lens.tolist() == [T + 3] * B

    def spin(y, weight):
        y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
        angle = torch.arange(T + 3, dtype=torch.float64)[:, None, None] * rotary.freq.cpu()
        a, b = y[..., :dim // 2], y[..., dim // 2:]
        return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1)

    xd = x.double()
    qd, kd, vd = spin(xd[:, :, :nq], w[0]), spin(xd[:, :, nq:nq + nkv], w[1]), xd[:, :, nq + nkv:]
    for t, got in zip(range(T, T + 3), outs):
        s = torch.einsum("bjd,bxjd->bjx", qd[:, t], kd[:, :t + 1].repeat_interleave(2, 2)) / dim ** 0.5
        p = torch.softmax(s, -1)
        want = torch.einsum("bjx,bxjd->bjd", p, vd[:, :t + 1].repeat_interleave(2, 2))
        # q and k rounded to bf16 (2^-8 each of themselves): scores off by scale * 2 * 2^-8 sum |q k|, probabilities by twice that, then the output's rounding
        ds = torch.einsum("bjd,bxjd->bjx", qd[:, t].abs(), kd[:, :t + 1].repeat_interleave(2, 2).abs()).amax(-1, keepdim=True) / dim ** 0.5 * (2.0 ** -7 + 2.0 ** -12)
        size = torch.einsum("bjx,bxjd->bjd", p, vd[:, :t + 1].repeat_interleave(2, 2).abs())
        near(got[:, 0], want, 2.0 ** -8 * want.abs() + (2 * ds + 2.0 ** -12) * size, f"step {t}")
