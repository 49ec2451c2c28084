"""The paged key/value cache operators against a plain implementation in 64 bits (GPU).

Tolerances, from the kernels' arithmetic (u = unit roundoff of the cache's type: 2^-24, 2^-11, 2^-8).
A score s = scale * sum q_i k_i is exact products summed in f32 (f32 caches: three products of split
operands, 2^-21 each): its error is at most ds = scale * sum |q_i k_i| * 2^-18 + |s| * 2^-21. Each probability
then has a relative error of at most 2 ds + 2^-20 (exponential, sum), plus u where it is rounded to
the cache's type, so an output is off by at most u |o| + (u_p + 2 ds + 2^-18) * sum p |v|; lse by ds + 2^-20 (1 + |lse|);
an accumulated weight w by (ds + 2^-18) w + 2^-23 |acc|. Copies and selections are exact."""
import math

import pytest
import torch

from technograd_b200 import _lib, kvcache

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
UNIT = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
INF = math.inf


class Case:
    """A cache with randomly placed pages. Rows that no position uses hold NaN."""

    def __init__(self, lens, nkv=2, group=2, dim=128, page=16, order="head", dtype=BF16, tokens=1, seed=1, spare=0, room=0):
        g = torch.Generator().manual_seed(seed)
        B = len(lens)
        self.lens, self.nkv, self.group, self.dim, self.page, self.dtype, self.T = lens, nkv, group, dim, page, dtype, tokens
        need = [-(-(n + room) // page) for n in lens]
        total, cols = sum(need) + 1 + spare, max(need) + 1
        place = torch.randperm(total, generator=g)
        table = torch.full((B, cols), -7, dtype=torch.int32)
        at = 0
        for b, w in enumerate(need):
            table[b, :w] = place[at:at + w].int()
            at += w
        self.free = place[at:]
        shape = (total, nkv, page, dim) if order == "head" else (total, page, nkv, dim)
        pools = [torch.full(shape, math.nan, dtype=dtype, device="cuda") for _ in range(2)]
        self.pk, self.pv = (x if order == "head" else x.transpose(1, 2) for x in pools)
        self.k = [torch.randn(n, nkv, dim, generator=g).to(dtype) for n in lens]
        self.v = [torch.randn(n, nkv, dim, generator=g).to(dtype) for n in lens]
        for b, n in enumerate(lens):
            p = torch.arange(n)
            where = table[b][p // page].long().cuda(), slice(None), (p % page).cuda()
            self.pk[where], self.pv[where] = self.k[b].cuda(), self.v[b].cuda()
        self.table, self.len = table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.cache = kvcache.PagedKV(self.pk, self.pv, self.table, self.len, max_len=max(lens))
        nq = nkv * group
        self.q = (2 * torch.randn(B, tokens, nq, dim, generator=g)).to(dtype)
        self.kn, self.vn = (torch.randn(B, tokens, nkv, dim, generator=g).to(dtype) for _ in range(2))

    def row(self, pool, b, h, p):
        return pool[int(self.table[b, p // self.page]), h, p % self.page]


def bits(rows):
    return torch.tensor([[x - (1 << 64) if x >> 63 else x for x in r] for r in rows], dtype=torch.int64)


def plain(c, mask=None, count=None, scale=None):
    """out, lse and their tolerances, and the probabilities [b][nq][t][x] with their tolerance, in 64 bits."""
    B, T, G = len(c.lens), c.T, c.group
    nq, scale = c.nkv * G, scale if scale is not None else c.dim ** -0.5
    out, lse = torch.zeros(B, T, nq, c.dim, dtype=torch.float64), torch.full((B, T, nq), -INF, dtype=torch.float64)
    tout, tlse, ps = torch.zeros_like(out), torch.zeros_like(lse), []
    up = 0 if c.dtype is F32 else UNIT[c.dtype]
    for b in range(B):
        m = count[b] if count else T
        k = torch.cat([c.k[b], c.kn[b, :m]]).double().cuda()
        v = torch.cat([c.v[b], c.vn[b, :m]]).double().cuda()
        n = c.lens[b]
        see = torch.ones(T, n + m, dtype=torch.bool)
        for t in range(T):
            for u in range(m):
                see[t, n + u] = (u <= t) if mask is None else bool(int(mask[b, t]) >> u & 1)
        see[m:] = False
        see = see.cuda()
        pb = []
        for j in range(nq):
            q, kk, vv = c.q[b, :, j].double().cuda(), k[:, j // G], v[:, j // G]
            kk, vv = torch.nan_to_num(kk, 0, 0, 0), torch.nan_to_num(vv, 0, 0, 0)
            s = (q @ kk.T * scale).masked_fill(~see, -INF)
            ds = (q.abs() @ kk.abs().T * scale * 2.0 ** -18 + torch.nan_to_num(s, 0, 0, 0).abs() * 2.0 ** -21).masked_fill(~see, 0)
            ds = ds.max(1).values if n + m else torch.zeros(T, dtype=torch.float64, device="cuda")
            z = torch.logsumexp(s, 1) if n + m else torch.full((T,), -INF, dtype=torch.float64, device="cuda")
            p = torch.nan_to_num(torch.exp(s - z[:, None]), 0)
            o, a = p @ vv, p @ vv.abs()
            out[b, :, j], lse[b, :, j] = o.cpu(), z.cpu()
            tout[b, :, j] = (UNIT[c.dtype] * o.abs() + (up + 2 * ds[:, None] + 2.0 ** -18) * a).cpu()
            tlse[b, :, j] = (ds + 2.0 ** -20 * (1 + torch.nan_to_num(z, 0, 0, 0).abs())).cpu()
            pb.append((p.cpu(), (p * (ds[:, None] + 2.0 ** -18)).cpu()))
        ps.append(pb)
    return out, lse, tout, tlse, ps


def near(got, want, tol, what):
    got = got.double().cpu()
    gone = torch.isinf(want)
    assert torch.equal(got[gone], want[gone]), what
    off = (got - want).abs()[~gone] - tol[~gone] - 1e-30
    assert not torch.isnan(got).any() and (off.numel() == 0 or off.max() <= 0), f"{what}: {off.max().item():.3g} over its tolerance"


def attend(c, mask=None, count=None, **kw):
    dev = dict(mask=None if mask is None else mask.cuda(), count=None if count is None else torch.tensor(count, dtype=torch.int32, device="cuda"))
    return kvcache.tree_attention(c.cache, c.q.cuda(), c.kn.cuda(), c.vn.cuda(), **dev, **kw)


def check_attend(c, mask=None, count=None):
    out, lse = attend(c, mask, count)
    want = plain(c, mask, count)
    near(out, want[0], want[2], "out")
    near(lse, want[1], want[3], "lse")
    return out, lse, want


def random_mask(B, T, seed, empty=True):
    g = torch.Generator().manual_seed(seed)
    m = [[int(torch.randint(0, 1 << 62, (1,), generator=g)) * 4 + t for t in range(T)] for _ in range(B)]
    return bits([[0 if empty and t % 5 == 2 else x & ((1 << T) - 1) for t, x in enumerate(r)] for r in m])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [8, 64, 80, 128, 136, 256])
@pytest.mark.parametrize("tokens,nkv,group", [(1, 2, 2), (7, 1, 3), (33, 2, 1), (64, 1, 4)])
def test_attention_shapes(cuda, dtype, dim, tokens, nkv, group):
    c = Case([70, 0, 1, 259], nkv, group, dim, 16, "head", dtype, tokens)
    check_attend(c, random_mask(4, tokens, 3), [tokens, tokens, (tokens + 1) // 2, 0])


@pytest.mark.parametrize("page,order", [(1, "pos"), (3, "head"), (5, "pos"), (16, "pos"), (24, "head"), (64, "pos"), (128, "head"), (1000, "pos")])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_pages(cuda, page, order, dtype):
    check_attend(Case([15, 16, 17, 63, 64, 65, 127, 300], 2, 2, 128, page, order, dtype, 5))


@pytest.mark.parametrize("lens", [[0], [1], [31], [1025], [4097, 3], [20011], [0, 0, 9000], [700] * 40])
@pytest.mark.parametrize("dtype,tokens,group", [(F32, 1, 2), (F16, 3, 8), (BF16, 64, 2), (BF16, 1, 1)])
def test_attention_lengths(cuda, lens, dtype, tokens, group):
    check_attend(Case(lens, 2, group, 64, 24, "head", dtype, tokens), random_mask(len(lens), tokens, 5))


def test_attention_many_heads_and_queries(cuda):
    check_attend(Case([333, 77], 3, 20, 64, 16, "pos", BF16, 64), random_mask(2, 64, 6))
    check_attend(Case([333, 77], 1, 71, 64, 16, "pos", F16, 2))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens", [4, 40])
def test_masked_rows_may_hold_anything(cuda, dtype, tokens):
    """Infinities and NaN in drafted rows reach only the tokens that see them, and rows past the
    count nobody."""
    c = Case([21, 0, 400], 2, 2, 128, 16, "head", dtype, tokens)
    bad = [1, tokens - 1]
    mask = random_mask(3, tokens, 8)
    mask &= ~((1 << bad[0]) | (1 << bad[1]))
    for x, y in ((c.kn, math.nan), (c.vn, INF)):
        x[:, bad[0]] = y
        x[:, bad[1]] = -INF if y == INF else y
    count = [tokens, tokens, tokens - 1]
    check_attend(c, mask, count)
    seen = mask.clone()
    seen[:, 0] |= 1 << bad[0]
    out, lse = attend(c, seen, count)
    want = plain(c, mask, count)
    assert torch.isnan(out[:, 0].float()).all() and torch.isnan(lse[:, 0]).all()
    near(out[:, 1:], want[0][:, 1:], want[2][:, 1:], "out")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens", [2, 48])
def test_infinite_values_of_seen_rows(cuda, dtype, tokens):
    """An infinite value of a seen row gives an infinite output to the tokens that see it, and only to them."""
    c = Case([300], 1, 2, 64, 16, "head", dtype, tokens)
    c.vn[0, 0, 0, 5] = INF
    mask = bits([[1 if t == 1 else 0 for t in range(tokens)]])
    out, _ = attend(c, mask)
    assert torch.isinf(out[0, 1, :, 5].float()).all() and torch.isfinite(out[0, 0].float()).all()
    assert torch.isfinite(out[0, 1, :, :5].float()).all() and torch.isfinite(out[0, 2:].float()).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_scores_far_apart(cuda, dtype):
    """Scores up to thousands: the running maximum rises late and by much; and scores all alike."""
    c = Case([500, 80], 2, 2, 64, 16, "head", dtype, 3)
    c.q *= 60
    check_attend(c)
    c.q *= 0
    check_attend(c)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_strided_operands(cuda, dtype):
    """q, k and v as slices of one projection's output, heads before tokens; a scale of one's own."""
    c = Case([100, 37], 2, 4, 64, 16, "head", dtype, 6)
    B, T, nq, D = c.q.shape
    x = torch.empty(B, T, (nq + 2 * c.nkv) * D + 8, dtype=dtype, device="cuda")
    q, k, v = (x[..., a * D:(a + w) * D].unflatten(2, (w, D)) for a, w in ((0, nq), (nq, c.nkv), (nq + c.nkv, c.nkv)))
    q.copy_(c.q), k.copy_(c.kn), v.copy_(c.vn)
    out, lse = kvcache.tree_attention(c.cache, q, k, v, scale=0.3)
    want = plain(c, scale=0.3)
    near(out, want[0], want[2], "out")
    near(lse, want[1], want[3], "lse")
    q2, k2, v2 = (y.transpose(1, 2).contiguous().transpose(1, 2) for y in (q, k, v))
    again = kvcache.tree_attention(c.cache, q2, k2, v2, scale=0.3)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


def test_offsets_past_32_bits(cuda):
    """A pool of more than 2^32 bytes whose used pages lie at its end."""
    c = Case([130], 1, 2, 128, 64, "head", BF16, 3, room=3)
    pages = (1 << 32) // (64 * 128 * 2) + 40
    pk, pv = (torch.zeros(pages, 1, 64, 128, dtype=BF16, device="cuda") for _ in range(2))
    where = torch.tensor([[pages - 1, pages - 30, pages - 7, pages - 3]], dtype=torch.int32, device="cuda")
    for i in range(3):
        pk[where[0, i]], pv[where[0, i]] = c.pk[c.table[0, i]], c.pv[c.table[0, i]]
    c.pk, c.pv, c.table = pk, pv, where
    c.cache = kvcache.PagedKV(pk, pv, where, c.len, max_len=130)
    out, lse, want = check_attend(c)
    got, fresh = kvcache.attention_weights(c.cache, c.q.cuda(), c.kn.cuda(), lse)
    assert abs(got.sum().item() + fresh.sum().item() - 6) < 1e-4
    n = kvcache.commit(c.cache, c.kn.cuda(), c.vn.cuda(), torch.tensor([3], dtype=torch.int32, device="cuda"))
    assert n.item() == 133 and torch.equal(pk[pages - 7, 0, 2:5].cpu(), c.kn[0, :, 0])
    dst = kvcache.PagedKV(pk, pv, torch.tensor([[pages - 2]], dtype=torch.int32, device="cuda"), torch.zeros_like(c.len), max_len=0)
    keep, _, _ = kvcache.evict(c.cache, dst, got, 64, recent=8)
    assert torch.equal(pv[pages - 2, 0].cpu(), c.v[0][keep[0, 0].long().cpu(), 0])


def test_another_stream_and_again(cuda):
    """Calls on a side stream, several in flight, give the same bits as calls on the default one."""
    cs = [Case([5000, 2000], 2, 2, 128, 16, "head", dt, t, seed=s) for s, (dt, t) in enumerate([(BF16, 1), (F32, 2), (F16, 40)])]
    args = [(c.cache, c.q.cuda(), c.kn.cuda(), c.vn.cuda()) for c in cs]
    want = [kvcache.tree_attention(*a) for a in args]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for s in (s1, s2, s1, s2):
        with torch.cuda.stream(s):
            got.append([kvcache.tree_attention(*a) for a in args])
    torch.cuda.synchronize()
    for g in got:
        for x, y in zip(g, want):
            assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


def test_in_a_graph(cuda):
    c = Case([900, 300], 2, 2, 128, 16, "head", BF16, 4)
    q, k, v = c.q.cuda(), c.kn.cuda(), c.vn.cuda()
    want = kvcache.tree_attention(c.cache, q, k, v)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = kvcache.tree_attention(c.cache, q, k, v)
    got[0].zero_(), got[1].zero_()
    g.replay()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- attention weights ---------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens,nkv,group,dim,page,tokens", [([1], 1, 1, 8, 5, 1), ([70, 0, 1, 259], 2, 2, 128, 16, 1), ([300, 64], 1, 8, 80, 24, 9),
                                                          ([129, 1000], 2, 3, 256, 3, 33), ([513], 1, 4, 64, 64, 64), ([0], 2, 2, 64, 16, 7)])
def test_weights(cuda, dtype, lens, nkv, group, dim, page, tokens):
    c = Case(lens, nkv, group, dim, page, "pos", dtype, tokens)
    B = len(lens)
    mask, count = random_mask(B, tokens, 4), [max(1, tokens - b) for b in range(B)]
    out, lse, want = check_attend(c, mask, count)
    g = torch.Generator().manual_seed(9)
    select = torch.randint(-(1 << 62), 1 << 62, (B,), generator=g) if tokens > 1 else torch.full((B,), 1)
    acc = torch.rand(B, nkv, max(lens) + 3, generator=g)
    exact_lse = want[1].float().cuda()  # the definition's own, so that the two do not differ by it
    for sel, a in ((select, acc), (None, None)):
        got, fresh = kvcache.attention_weights(c.cache, c.q.cuda(), c.kn.cuda(), exact_lse, mask.cuda(),
                                               torch.tensor(count, dtype=torch.int32, device="cuda"),
                                               None if sel is None else sel.cuda(), None if a is None else a.cuda())
        assert got.shape == (B, nkv, max(lens)) and fresh.shape == (B, nkv, tokens)
        for b in range(B):
            n, m = lens[b], count[b]
            on = torch.tensor([(1 if sel is None else int(sel[b]) >> t & 1) for t in range(tokens)], dtype=torch.float64)
            lse_off = (want[1][b].float().double() - want[1][b]).abs()  # rounding of the lse it was given
            for h in range(nkv):
                w, tol = torch.zeros(n + m, dtype=torch.float64), torch.zeros(n + m, dtype=torch.float64)
                for j in range(h * group, (h + 1) * group):
                    p, tp = want[4][b][j]
                    w += on @ p
                    tol += on @ (tp + 2 * p * torch.nan_to_num(lse_off[:, j], 0, 0, 0)[:, None])
                base = a[b, h, :n].double() if a is not None else torch.zeros(n, dtype=torch.float64)
                near(got[b, h, :n], base + w[:n], tol[:n] + 2.0 ** -23 * (base + w[:n]), "acc")
                near(fresh[b, h, :m], w[n:], tol[n:] + 1e-30, "new")
                assert not got[b, h, n:].any() and not fresh[b, h, m:].any()


def test_weights_in_place_and_masked_rows(cuda):
    """acc may be updated in place; a drafted key that nobody sees may hold NaN."""
    c = Case([200, 31], 2, 2, 64, 16, "head", BF16, 3)
    c.kn[:, 2] = math.nan
    mask = bits([[1, 3, 0], [0, 0, 3]])
    q, kn, vn = c.q.cuda(), c.kn.cuda(), torch.nan_to_num(c.vn).cuda()
    _, lse = kvcache.tree_attention(c.cache, q, kn, vn, mask.cuda())
    one, fresh = kvcache.attention_weights(c.cache, q, kn, lse, mask.cuda())
    assert torch.isfinite(one).all() and torch.isfinite(fresh).all() and not fresh[:, :, 2].any()
    total = one.sum(2) + fresh.sum(2)  # each row that sees something spreads a weight of 1
    assert torch.allclose(total, torch.tensor([[6.0], [6.0]], device="cuda").expand(2, 2), atol=1e-4)
    acc = one.clone()
    two, _ = kvcache.attention_weights(c.cache, q, kn, lse, mask.cuda(), acc=acc)
    m = mask.cuda()
    drafts = kvcache._drafts(c.cache, q, kn, None, m, None, None)
    fresh2 = torch.empty_like(fresh)
    _lib.check(cuda.tg_cuda_attn_weights(c.cache._at, drafts, lse.data_ptr(), None, acc.data_ptr(), acc.stride(0), acc.stride(1),
                                         acc.data_ptr(), fresh2.data_ptr(), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(acc, two) and torch.equal(fresh, fresh2)


# ---- commit and evict ----------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim,page,order,tokens", [(8, 5, "head", 1), (128, 16, "pos", 9), (80, 3, "head", 64), (256, 64, "pos", 300)])
def test_commit(cuda, dtype, dim, page, order, tokens):
    lens = [0, 33, 64, 7]
    c = Case(lens, 3, 1, dim, page, order, dtype, tokens, room=tokens)
    count = [tokens, tokens // 2, 0, min(1, tokens)]
    g = torch.Generator().manual_seed(2)
    path = torch.stack([torch.randperm(tokens, generator=g) for _ in lens]).int()
    for b, m in enumerate(count):
        path[b, m:] = -5  # not looked at
    new, acc = torch.rand(4, 3, tokens, generator=g), torch.rand(4, 3, max(lens) + tokens, generator=g)
    for p in (path, None):
        before = c.pk.clone(), c.pv.clone()
        got = acc.cuda()
        n = kvcache.commit(c.cache, c.kn.cuda(), c.vn.cuda(), torch.tensor(count, dtype=torch.int32, device="cuda"),
                           None if p is None else p.cuda(), new.cuda(), got)
        assert n.tolist() == [a + b for a, b in zip(lens, count)]
        want, (wk, wv) = acc.clone(), before
        for b, m in enumerate(count):
            for i in range(m):
                f, at = (i if p is None else int(p[b, i])), lens[b] + i
                wk[int(c.table[b, at // page]), :, at % page] = c.kn[b, f].cuda()
                wv[int(c.table[b, at // page]), :, at % page] = c.vn[b, f].cuda()
                want[b, :, at] = new[b, :, f]
        assert torch.equal(got.cpu(), want)
        for x, y in ((c.pk, wk), (c.pv, wv)):
            assert torch.equal(torch.nan_to_num(x.float(), 777), torch.nan_to_num(y.float(), 777))


def plain_keep(acc, n, budget, recent, sink):
    if n <= budget:
        return list(range(n))
    key = [-INF if math.isnan(x) else x for x in acc]
    low = [math.isnan(x) for x in acc]
    mid = sorted(range(sink, n - recent), key=lambda i: (low[i], -key[i], i))[:budget - sink - recent]
    return sorted(list(range(sink)) + mid + list(range(n - recent, n)))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens,dim,page,order,budget,recent,sink", [
    ([300, 0, 1, 64, 65], 128, 16, "head", 64, 10, 4), ([301, 299], 8, 5, "pos", 200, 31, 4), ([5000, 1025], 64, 64, "head", 1024, 0, 0),
    ([40, 90], 80, 24, "pos", 30, 30, 0), ([40, 90], 80, 1, "pos", 30, 0, 30), ([2049], 256, 3, "head", 1, 0, 0), ([100], 128, 16, "head", 300, 7, 3),
    ([70000], 8, 64, "head", 33000, 100, 4)])
@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
def test_evict(cuda, dtype, lens, dim, page, order, budget, recent, sink, kind):
    c = Case(lens, 2, 1, dim, page, order, dtype, 1, spare=len(lens) * (-(-budget // page)))
    g = torch.Generator().manual_seed(11)
    acc = torch.randn(len(lens), 2, max(lens) + 5, generator=g)
    if kind == "ties":
        acc = (acc * 2).round() / 2
    if kind == "odd":
        odd = torch.tensor([math.nan, -math.nan, INF, -INF, 0.0, -0.0, 1e-45, -1e-45, 3.4e38, -3.4e38])
        acc = odd[torch.randint(0, 10, acc.shape, generator=g)]
    cols = -(-budget // page)
    table = c.free[:len(lens) * cols].view(len(lens), cols).int().cuda()
    dst = kvcache.PagedKV(c.pk, c.pv, table, torch.zeros_like(c.len), max_len=0)
    keep, out, n = kvcache.evict(c.cache, dst, acc.cuda(), budget, recent, sink)
    assert n.tolist() == [min(x, budget) for x in lens]
    for b in range(len(lens)):
        for h in range(2):
            want = plain_keep(acc[b, h, :lens[b]].tolist(), lens[b], budget, recent, sink)
            assert keep[b, h].tolist() == want + [-1] * (budget - len(want))
            w = torch.tensor(want, dtype=torch.long)
            assert torch.equal(torch.nan_to_num(out[b, h, :len(want)].cpu(), 777), torch.nan_to_num(acc[b, h][w], 777)) and not out[b, h, len(want):].any()
            i = torch.arange(len(want))
            at = table[b].cpu()[i // page].long().cuda(), h, (i % page).cuda()
            assert torch.equal(c.pk[at].cpu(), c.k[b][w, h]) and torch.equal(c.pv[at].cpu(), c.v[b][w, h])
    more, _, _ = kvcache.evict(c.cache, dst, acc.cuda(), budget, recent, sink)
    assert torch.equal(more, keep)


# ---- refusals and reports ------------------------------------------------------------------------------

def test_refusals(cuda):
    c = Case([40, 20], 2, 2, 64, 16, "head", BF16, 3)
    q, k, v = c.q.cuda(), c.kn.cuda(), c.vn.cuda()
    mask, count = torch.zeros(2, 3, dtype=torch.int64, device="cuda"), torch.tensor([3, 3], dtype=torch.int32, device="cuda")
    for bad in (dict(q=q.float()), dict(k=k.float()), dict(v=v[:, :2]), dict(q=q[:, :2]), dict(q=q.cpu()), dict(mask=mask[:1]), dict(mask=mask.int()),
                dict(count=count.long()), dict(k=k.transpose(2, 3).contiguous().transpose(2, 3)), dict(k=k[:1], v=v[:1]), dict(v=v.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            kvcache.tree_attention(**{**dict(cache=c.cache, q=q, k=k, v=v, mask=mask, count=count), **bad})
    wide = torch.zeros(2, 65, 4, 64, dtype=BF16, device="cuda")
    odd = torch.zeros(2, 3, 4, 65, dtype=BF16, device="cuda")[..., 1:]
    for args in ((wide, wide[:, :, :2], wide[:, :, :2]), (q[:, :, :3], k, v), (odd, k, v), (q, odd[:, :, :2], odd[:, :, :2])):
        with pytest.raises(_lib.TgCudaError) as e:
            kvcache.tree_attention(c.cache, *args)
        assert e.value.status == _lib.EINVAL
    with pytest.raises(ValueError):
        kvcache.PagedKV(c.pk, c.pv.float(), c.table, c.len)
    with pytest.raises(ValueError):
        kvcache.PagedKV(c.pk, c.pv, c.table.long(), c.len)
    for kw in (dict(max_len=10 ** 6), dict(max_len=-1)):
        with pytest.raises(_lib.TgCudaError):
            kvcache.tree_attention(kvcache.PagedKV(c.pk, c.pv, c.table, c.len, **kw), q, k, v)
    lse, acc = torch.zeros(2, 3, 4, device="cuda"), torch.zeros(2, 2, 40, device="cuda")
    for bad in (dict(lse=lse[:, :2]), dict(acc=acc[:, :, :39]), dict(acc=acc.double()), dict(select=count)):
        with pytest.raises(ValueError):
            kvcache.attention_weights(**{**dict(cache=c.cache, q=q, k=k, lse=lse, acc=acc), **bad})
    with pytest.raises(ValueError):
        kvcache.commit(c.cache, k, v, count, new=torch.zeros(2, 2, 3, device="cuda"))
    with pytest.raises(ValueError):
        kvcache.commit(c.cache, k, v, count, path=count)
    for bad in (dict(budget=0), dict(acc=acc[:, :1])):
        with pytest.raises(ValueError):
            kvcache.evict(**{**dict(cache=c.cache, dst=c.cache, acc=acc, budget=8), **bad})
    for kw in (dict(recent=9), dict(sink=-1), dict(recent=5, sink=4)):
        with pytest.raises(_lib.TgCudaError):
            kvcache.evict(c.cache, c.cache, acc, 8, **kw)


def reported(f):
    torch.cuda.synchronize()
    with pytest.raises(_lib.TgCudaError) as e:
        f()
    assert e.value.status == _lib.EDEVICE
    f()  # reported once
    torch.cuda.synchronize()
    return str(e.value)


def test_device_data_out_of_range_is_reported(cuda):
    """Bad lengths, page numbers and paths are not followed: the call completes and a later one says so."""
    c = Case([40, 20], 2, 2, 64, 16, "head", BF16, 3)
    q, k, v = c.q.cuda(), c.kn.cuda(), c.vn.cuda()
    good = lambda: kvcache.tree_attention(c.cache, q, k, v)  # noqa: E731
    for at, bad in ((0, 10 ** 6), (2, -1)):
        t = c.table.clone()
        t[0, at] = bad
        out, _ = kvcache.tree_attention(kvcache.PagedKV(c.pk, c.pv, t, c.len, max_len=40), q, k, v)
        assert torch.isfinite(out.float()).all()
        assert "page number" in reported(good)
    for bad in ([41, 20], [40, -3]):
        n = torch.tensor(bad, dtype=torch.int32, device="cuda")
        out, _ = kvcache.tree_attention(kvcache.PagedKV(c.pk, c.pv, c.table, n, max_len=40), q, k, v)
        assert "len" in reported(good)
    n = torch.tensor([3, 3], dtype=torch.int32, device="cuda")
    room = kvcache.PagedKV(c.pk, c.pv, c.table[:, :2].contiguous(), torch.tensor([31, 20], dtype=torch.int32, device="cuda"), max_len=32)
    kvcache.commit(room, k, v, n)
    assert "past the table" in reported(good)
    kvcache.commit(c.cache.with_lens(torch.tensor([0, 0], dtype=torch.int32, device="cuda"), 40), k, v, n, path=torch.full((2, 3), 3, dtype=torch.int32, device="cuda"))
    assert "path" in reported(good)


@pytest.mark.parametrize("lens,nkv,budget,recent,sink,kind", [
    ([131072], 1, 4000, 100, 4, "random"), ([131071, 40000], 2, 60000, 0, 0, "ties"), ([100000], 1, 5, 2, 3, "random"), ([450001], 1, 70000, 9, 1, "random"),
    ([60000], 1, 59999, 0, 0, "same"), ([9000] * 3, 1, 4500, 0, 0, "same"), ([30000], 1, 29000, 0, 0, "nan")])
def test_evict_long(cuda, lens, nkv, budget, recent, sink, kind):
    """Heads whose weights span several CTAs, fit no shared memory, or are all alike."""
    c = Case(lens, nkv, 1, 8, 64, "head", BF16, 1, spare=len(lens) * (-(-budget // 64)))
    g = torch.Generator().manual_seed(12)
    acc = torch.rand(len(lens), nkv, max(lens), generator=g)
    if kind == "ties":
        acc = (acc * 50).floor() / 50
    if kind == "same":
        acc[:] = 0.25
    if kind == "nan":
        acc[:, :, 100:] = math.nan
    cols = -(-budget // 64)
    dst = kvcache.PagedKV(c.pk, c.pv, c.free[:len(lens) * cols].view(len(lens), cols).int().cuda(), torch.zeros_like(c.len), max_len=0)
    keep, out, _ = kvcache.evict(c.cache, dst, acc.cuda(), budget, recent, sink)
    for b, n in enumerate(lens):
        for h in range(nkv):
            want = plain_keep(acc[b, h, :n].tolist(), n, budget, recent, sink)
            assert keep[b, h].tolist() == want + [-1] * (budget - len(want))
            w = torch.tensor(want)
            assert torch.equal(torch.nan_to_num(out[b, h, :len(want)].cpu(), 7), torch.nan_to_num(acc[b, h][w], 7))
            i = torch.arange(len(want))
            at = dst.table[b].cpu()[i // 64].long().cuda(), h, (i % 64).cuda()
            assert torch.equal(c.pk[at].cpu(), c.k[b][w, h]) and torch.equal(c.pv[at].cpu(), c.v[b][w, h])


@pytest.mark.parametrize("page,order", [(8, "head"), (16, "pos"), (32, "head"), (64, "pos"), (128, "head"), (192, "pos"), (256, "head"), (40, "pos"), (4, "head")])
@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (BF16, 72)])
def test_many_rows_over_pages(cuda, page, order, dtype, dim):
    """Tiles of many rows read pages in boxes or row by row; what lies past a sequence's end is NaN."""
    c = Case([1, 127, 128, 129, 700, 0], 2, 3, dim, page, order, dtype, 33)
    mask = random_mask(6, 33, 7)
    out, lse, want = check_attend(c, mask)
    acc, fresh = kvcache.attention_weights(c.cache, c.q.cuda(), c.kn.cuda(), want[1].float().cuda(), mask.cuda())
    rows = (want[1] > -INF).sum(1).view(6, 2, 3).sum(2)  # each row that sees something spreads a weight of 1
    assert (acc.sum(2).cpu() + fresh.sum(2).cpu() - rows).abs().max() < 1e-3


def test_negative_and_zero_scale(cuda):
    for tokens in (2, 40):
        c = Case([300, 9], 2, 2, 128, 16, "head", BF16, tokens)
        for scale in (-0.1, 0.0):
            out, lse = attend(c, scale=scale)
            flip = Case([300, 9], 2, 2, 128, 16, "head", BF16, tokens)
            flip.q = -flip.q if scale < 0 else flip.q * 0
            want = plain(flip, scale=abs(scale) or 0.1)
            near(out, want[0], want[2], "out")
            near(lse, want[1], want[3], "lse")


def test_f32_sums_over_many_keys_do_not_drift(cuda):
    """60000 keys: products rounded to nearest keep the output within sqrt(steps) * 2^-24 of the definition (about
    2^-19 here); sums that truncate would be off by 2^-16."""
    c = Case([60000], 1, 4, 64, 64, "head", F32, 2)
    c.q *= 0.25
    out, lse = attend(c)
    want = plain(c)
    assert ((out.cpu().double() - want[0]).norm() / want[0].norm()).item() < 2.0 ** -18
    assert (lse.cpu().double() - want[1]).abs().max() < 2.0 ** -20 * 16


@pytest.mark.parametrize("dim", [4, 64, 68, 128, 252, 256])
@pytest.mark.parametrize("tokens,nkv,group", [(1, 2, 1), (1, 1, 3), (2, 2, 2), (5, 1, 1), (2, 1, 4), (3, 1, 3), (4, 1, 4)])
def test_f32_with_few_rows(cuda, dim, tokens, nkv, group):
    """1 to 16 rows per key head, on the FMA units up to 8."""
    for lens in ([70, 0, 1, 259], [2000]):
        c = Case(lens, nkv, group, dim, 16, "pos", F32, tokens)
        check_attend(c, random_mask(len(lens), tokens, 3), [tokens, tokens, (tokens + 1) // 2, 0][:len(lens)])


def test_weights_take_any_strides(cuda):
    """lse, q and k as views whose rows or tokens are not next to each other; acc as a slice of something wider."""
    c = Case([150, 41], 1, 2, 64, 16, "head", BF16, 5)
    q, kn, vn = c.q.cuda(), c.kn.cuda(), c.vn.cuda()
    _, lse = kvcache.tree_attention(c.cache, q, kn, vn)
    wide = torch.rand(2, 3, 200, device="cuda")
    want = kvcache.attention_weights(c.cache, q, kn, lse, acc=wide[:, 1:2].contiguous())
    turned = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, kn, lse)]
    got = kvcache.attention_weights(c.cache, *turned, acc=wide[:, 1:2])
    assert not turned[2].is_contiguous() and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
