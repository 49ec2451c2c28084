"""The paged key/value cache operators where their kernels' parts meet: short units next to each other, several CTAs on one
head, few rows of a block (GPU). Cases, definitions in 64 bits and tolerances as in test_gpu_kvcache.py, and half of f16's
least spacing (2^-24) more where an f16 output is below its normal numbers: u |o| is the rounding of normal ones only."""
import copy
import math

import pytest
import torch

from technograd_b200 import _lib, kvcache  # noqa: F401
from test_gpu_kvcache import BF16, F16, F32, INF, UNIT, Case, attend, bits, check_attend, near, plain, plain_keep, random_mask  # noqa: F401

pytestmark = pytest.mark.gpu


def check(got, want, dtype):
    """out and lse against plain()'s."""
    near(got[0], want[0], want[2] + (2.0 ** -25 if dtype is F16 else 0), "out")
    near(got[1], want[1], want[3], "lse")


def check_weights(c, mask=None, count=None, select=None, acc=None):
    """attention_weights key by key against plain()'s probabilities, given its lse rounded to f32."""
    want = plain(c, mask, count)
    lse = want[1].float()
    dev = [None if x is None else x.cuda() for x in (mask, None if count is None else torch.tensor(count, dtype=torch.int32), select, acc)]
    got, fresh = (x.cpu() for x in kvcache.attention_weights(c.cache, c.q.cuda(), c.kn.cuda(), lse.cuda(), *dev))
    for b, n in enumerate(c.lens):
        m = count[b] if count else c.T
        on = torch.tensor([1 if select is None else int(select[b]) >> t & 1 for t in range(c.T)], dtype=torch.float64)
        off = torch.nan_to_num((lse[b].double() - want[1][b]).abs(), 0, 0, 0)  # rounding of the lse it was given
        for h in range(c.nkv):
            w, tol = torch.zeros(n + m, dtype=torch.float64), torch.zeros(n + m, dtype=torch.float64)
            for j in range(h * c.group, (h + 1) * c.group):
                p, tp = want[4][b][j]
                w += on @ p
                tol += on @ (tp + 2 * p * off[:, j, None])
            base = torch.zeros(n, dtype=torch.float64) if acc is None else acc[b, h, :n].double()
            near(got[b, h, :n], base + w[:n], tol[:n] + 2.0 ** -23 * (base + w[:n]), "acc")
            near(fresh[b, h, :m], w[n:], tol[n:] + 2.0 ** -23 * w[n:], "fresh")
            assert not got[b, h, n:].any() and not fresh[b, h, m:].any()


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("lens", [[0] * 200 + [700], [0, 1, 128, 129] * 60, [128] * 300])
def test_short_units_after_each_other(cuda, lens, dtype, dim):
    """Many units of one or two tiles to a CTA of the 128-row kernel: each row's reference and sum are its own unit's. The
    rows' scores differ by hundreds from unit to unit, so that another unit's would show."""
    c = Case(lens, 2, 2, dim, 16, "head", dtype, 20)
    c.q *= torch.tensor([1.0, 20.0, 0.05])[torch.arange(len(lens)) % 3][:, None, None, None]
    mask = random_mask(len(lens), 20, 3)
    out, lse = attend(c, mask)
    check((out, lse), plain(c, mask), dtype)
    for _ in range(20):
        again = attend(c, mask)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("heads,n,want", [(1, 70000, 20000), (2, 20000, 7000), (70, 40000, 5000), (3, 140001, 1000)])
def test_evict_heads_of_several_ctas(cuda, heads, n, want):
    """Heads whose keys span a cluster of CTAs, next to heads that end before they count anything (all kept) and that
    compete for one place, many times over and beside other work."""
    lens = [n, want, want + 1][:heads] + [n] * (heads - 3)
    c = Case([1] * heads, 1, 1, 8, 64, "head", F32, 1)
    acc = torch.rand(heads, 1, n, generator=torch.Generator().manual_seed(5))
    src = kvcache.PagedKV(c.pk, c.pv, torch.zeros(heads, -(-n // 64), dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda"), max_len=n)
    cols = -(-want // 64)
    pool = torch.empty(heads * cols, 1, 64, 8, device="cuda")
    dst = kvcache.PagedKV(pool, torch.empty_like(pool), torch.arange(heads * cols, dtype=torch.int32, device="cuda").view(heads, cols), torch.zeros_like(src.lens), max_len=0)
    dev = acc.cuda()
    keep, out, _ = kvcache.evict(src, dst, dev, want, want // 8, 2)
    for b in range(0, heads, 1 if heads < 4 else 13):
        kept = plain_keep(acc[b, 0, :lens[b]].tolist(), lens[b], want, want // 8, 2)
        assert keep[b, 0, :len(kept)].tolist() == kept and torch.equal(out[b, 0, :len(kept)].cpu(), acc[b, 0, kept])
    side = torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(side):
            pool.new_empty(1 << 26).zero_()
        again, _, _ = kvcache.evict(src, dst, dev, want, want // 8, 2)
        assert torch.equal(again, keep)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens,group", [(1, 1), (1, 3), (3, 3), (13, 1), (18, 1)])
def test_join_of_blocks_with_few_rows(cuda, dtype, dim, tokens, group):
    """One long sequence: many partial results of rows that fill a block of the join only in part."""
    c = Case([9001], 1, group, dim, 64, "head", dtype, tokens)
    mask = random_mask(1, tokens, 4)
    check(attend(c, mask), plain(c, mask), dtype)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (F32, 128), (BF16, 256)])
@pytest.mark.parametrize("tokens,group", [(17, 1), (32, 1), (63, 5), (64, 5)])
def test_drafted_weights_of_all_tokens(cuda, dtype, dim, tokens, group):
    """A tile of keys may be wider than a mask: every drafted key has its own weight, the keys past the tokens none."""
    c = Case([40, 0, 3], 1, group, dim, 16, "head", dtype, tokens)
    check_weights(c, random_mask(3, tokens, 6), [tokens, tokens, tokens - 1])
    check_weights(c)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,group", [(2, 2), (9, 1), (9, 2), (40, 1), (40, 4)])
def test_keys_of_minus_infinity(cuda, dtype, tokens, group):
    """Keys of -infinity against positive queries have scores of -infinity: no weight, in the cache and among the drafted; a
    token that sees nothing else has 0 and -infinity."""
    c = Case([0, 5, 300], 2, group, 64, 16, "head", dtype, tokens)
    c.q[:] = c.q.abs() + 0.5
    gone = [torch.zeros(n, dtype=torch.bool) for n in c.lens]
    gone[1][:], gone[2][torch.arange(0, 300, 7)] = True, True
    for b, n in enumerate(c.lens):
        for p in gone[b].nonzero()[:, 0].tolist():
            c.pk[int(c.table[b, p // c.page]), :, p % c.page] = -INF
    c.kn[:, 1] = -INF
    mask = bits([[2 if t == 0 else (2 << t) - 1 for t in range(tokens)]] * 3)
    got = attend(c, mask)
    rest = copy.copy(c)
    rest.lens, rest.k, rest.v = [int((~x).sum()) for x in gone], [x[~y] for x, y in zip(c.k, gone)], [x[~y] for x, y in zip(c.v, gone)]
    want = plain(rest, mask & ~2)
    assert (want[1][:2, 0] == -INF).all()
    check(got, want, dtype)
    acc, fresh = kvcache.attention_weights(c.cache, c.q.cuda(), c.kn.cuda(), want[1].float().cuda(), mask.cuda())
    assert torch.isfinite(acc).all() and torch.isfinite(fresh).all() and not fresh[:, :, 1].any()
    for b, n in enumerate(c.lens):
        assert not acc[b, :, :n][:, gone[b].cuda()].any()
    rows = (want[1] > -INF).sum(1).view(3, 2, group).sum(2)
    assert (acc.sum(2).cpu() + fresh.sum(2).cpu() - rows).abs().max() < 1e-3  # each row that sees something spreads a weight of 1


def with_infinities(dtype, tokens, group):
    """Token 0's value row holds an infinity and a NaN. Masks: every token sees itself and token 0; and itself alone."""
    c = Case([0, 5, 300, 5000], 2, group, 64, 16, "head", dtype, tokens)
    c.q[:] = c.q.abs() + 0.5  # so that a key of -60 has a score of -240 or less, and one of 60 one of 240 or more
    c.vn[:, 0, :, 5], c.vn[:, 0, :, 6] = INF, math.nan
    return c, bits([[1 << t | 1 for t in range(tokens)]] * 4), bits([[1 << t for t in range(tokens)]] * 4)


ROWS = [(2, 2), (9, 2), (40, 1), (40, 2)]  # tokens and heads per key head: 4, 18, 40 and 80 rows


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,group", ROWS)
@pytest.mark.parametrize("far", [-60.0, -INF])
def test_infinities_of_no_weight(cuda, dtype, tokens, group, far):
    """A drafted row that a token sees with a probability of 0 in f32 adds nothing to it, whatever it holds."""
    c, mask, alone = with_infinities(dtype, tokens, group)
    c.kn[:, 0] = far
    got, want = attend(c, mask), plain(c, alone)
    check([x[:, 1:] for x in got], [x[:, 1:] for x in want[:4]], dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,group", ROWS)
def test_infinities_that_lose_their_weight(cuda, dtype, tokens, group):
    """... also where only a later key takes its probability away; token 0, which sees nothing else drafted, gets them."""
    c, mask, alone = with_infinities(dtype, tokens, group)
    c.kn[:, 0], c.kn[:, 1:] = 0, 60
    got, want = attend(c, mask), plain(c, alone)
    check([x[:, 1:] for x in got], [x[:, 1:] for x in want[:4]], dtype)
    out = got[0][:, 0].float()
    assert torch.isinf(out[..., 5]).all() and torch.isnan(out[..., 6]).all() and torch.isfinite(out[..., :5]).all() and torch.isfinite(out[..., 7:]).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,group", [(1, 2), (16, 2), (17, 2), (64, 4), (64, 5)])
def test_weights_of_large_scores(cuda, dtype, tokens, group):
    """Scores of thousands that f32 holds exactly: a weight is 2^((scale s - lse) log2 e), whose error follows the difference d
    and not the score: 2^-24 |d| for it, its product and log2 e each, 2^-22 of the exponential, 2^-24 for each row of the sum."""
    c = Case([150, 3], 1, group, 64, 16, "head", dtype, tokens)
    g = torch.Generator().manual_seed(3)
    c.q[:] = 0
    c.q[..., 0] = 128
    for b, n in enumerate(c.lens):
        c.k[b][:] = 0
        c.k[b][..., 0] = torch.randint(195, 201, (n, 1), generator=g).to(dtype)
        for p in range(n):
            c.pk[int(c.table[b, p // 16]), :, p % 16] = c.k[b][p].cuda()
    c.kn[:] = 0
    c.kn[..., 0] = torch.randint(195, 201, c.kn.shape[:3], generator=g).to(dtype)
    lse = 3200 + 2 * torch.rand(2, tokens, group, generator=g)
    acc, fresh = (x.cpu().double() for x in kvcache.attention_weights(c.cache, c.q.cuda(), c.kn.cuda(), lse.cuda(), scale=0.125))
    for b, n in enumerate(c.lens):
        k = torch.cat([c.k[b][:, 0, 0], c.kn[b, :, 0, 0]]).double()
        d = 16 * k[None, None] - lse[b].double()[:, :, None]  # [token][head][key]
        w = torch.exp(d)
        tol = w * (3 * 2.0 ** -24 * d.abs() + 2.0 ** -22 + 2.0 ** -24 * tokens * group)
        see = torch.ones(tokens, n + tokens)
        see[:, n:].tril_()
        w, tol = ((x * see[:, None]).sum((0, 1)) for x in (w, tol))
        near(acc[b, 0, :n], w[:n], tol[:n], "acc")
        near(fresh[b, 0], w[n:], tol[n:], "fresh")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens,group", [(1, 2), (4, 2), (3, 3), (16, 2), (20, 2), (64, 2)])
@pytest.mark.parametrize("sharp", [1, 4])
def test_16_bit_outputs_are_rounded_once(cuda, dtype, dim, tokens, group, sharp):
    """An output's error is its own rounding and that of an f32 softmax, whether many keys share the weight or one has most of it:
    probabilities keep 2^-15 (bf16) or 2^-20 (f16, with 2^-35 of the largest for each key, below its normal numbers) of theirs."""
    c = Case([1, 0, 300, 2000], 2, group, dim, 16, "head", dtype, tokens)
    c.q *= sharp
    mask = random_mask(4, tokens, 9, empty=False)
    got, want = attend(c, mask), plain(c, mask)
    of = copy.copy(c)
    of.v, of.vn = [x.abs() for x in c.v], c.vn.abs()
    spread = plain(of, mask)[0]  # sum p |v|
    kept = 2.0 ** -15 if dtype is BF16 else 2.0 ** -20
    tol = want[2] - (UNIT[dtype] - kept) * spread
    if dtype is F16:
        tol += 2.0 ** -25 + torch.tensor([(n + tokens) * 2.0 ** -35 * 6 for n in c.lens])[:, None, None, None]
    near(got[0], want[0], tol, "out")
    near(got[1], want[1], want[3], "lse")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,group", [(1, 2), (9, 1), (40, 1), (64, 2)])
def test_infinite_cached_values(cuda, dtype, tokens, group):
    """An infinite element of a cached value row with a probability (here 2^-14 or more) is infinite in the outputs, with its sign,
    and nothing else is, though a probability is two parts to the tensor core."""
    c = Case([200], 1, group, 64, 16, "head", dtype, tokens)
    c.q *= 0.25
    for i, p in enumerate((0, 17, 63, 64, 199)):
        for at, x in ((i, INF), (20 + i, -INF)):
            c.pv[int(c.table[0, p // 16]), 0, p % 16, at] = x
    for zero in (False, True):  # and all scores alike: probabilities of one bit
        out = attend(c)[0].float()
        assert (out[..., :5] == INF).all() and (out[..., 20:25] == -INF).all()
        assert torch.isfinite(out[..., 5:20]).all() and torch.isfinite(out[..., 25:]).all()
        c.q *= 0


def test_lengths_past_32_bits_are_refused(cuda):
    """A max_len of 2^32 + 40 is not one of 40, nor is a table that holds more positions than an int numbers."""
    c = Case([40], 1, 1, 64, 16, "head", BF16, 1)
    with pytest.raises(ValueError, match="32 bits"):
        kvcache.PagedKV(c.pk, c.pv, c.table, c.len, max_len=2 ** 32 + 40)
    page = torch.zeros(1, 1, 1 << 20, 8, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="32 bits"):
        kvcache.PagedKV(page, page, torch.zeros(1, 1 << 12, dtype=torch.int32, device="cuda"), c.len)


@pytest.mark.parametrize("page,order", [(8, "head"), (16, "pos"), (24, "pos"), (32, "head"), (64, "pos"), (128, "head"), (192, "pos"), (40, "pos"), (4, "head")])
@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (BF16, 72)])
@pytest.mark.parametrize("tokens,group", [(33, 3), (64, 4)])
def test_weights_of_every_key_over_pages(cuda, page, order, dtype, dim, tokens, group):
    """Key by key, which a tile's keys in another order would not pass: boxes of pages, their two halves of the dimensions, several
    heads; what lies past a sequence's end is NaN."""
    c = Case([1, 127, 129, 700, 0], 2, group, dim, page, order, dtype, tokens)
    check_weights(c, random_mask(5, tokens, 7), acc=torch.rand(5, 2, 700, generator=torch.Generator().manual_seed(1)))


def with_room(c, positions):
    """The same cache with a table for so many positions and max_len with it: calls are cut as for long sequences."""
    more = torch.full((len(c.lens), -(-positions // c.page)), -7, dtype=torch.int32, device="cuda")
    more[:, :c.table.shape[1]] = c.table
    c.cache = kvcache.PagedKV(c.pk, c.pv, more, c.len, max_len=positions)
    return c


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (BF16, 72), (F32, 64), (BF16, 256)])
@pytest.mark.parametrize("tokens,group", [(1, 2), (8, 2), (17, 1), (16, 2), (40, 1)])
@pytest.mark.parametrize("positions", [4096, 60000])
def test_attention_cut_for_long_sequences(cuda, dtype, dim, tokens, group, positions):
    """What a CTA has to do at most decides which kernel takes a call: the results are the definition's with each."""
    c = with_room(Case([500, 0, 129, 1, 128, 700, 64], 2, group, dim, 16, "head", dtype, tokens), positions)
    mask = random_mask(7, tokens, 3)
    check(attend(c, mask), plain(c, mask), dtype)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (BF16, 72), (F32, 64)])
@pytest.mark.parametrize("tokens,group", [(1, 1), (1, 2), (8, 2), (17, 1), (16, 2), (40, 1), (64, 4), (64, 5)])
@pytest.mark.parametrize("positions", [4096, 20000, 70000])
def test_weights_cut_for_long_sequences(cuda, dtype, dim, tokens, group, positions):
    """... and the weights', with what was there before and zeros past each sequence's end."""
    c = with_room(Case([500, 0, 129, 1, 128, 700, 64], 2, group, dim, 16, "head", dtype, tokens), positions)
    check_weights(c, random_mask(7, tokens, 3), acc=torch.rand(7, 2, positions, generator=torch.Generator().manual_seed(1)))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,group", [(1, 2), (16, 2), (32, 4), (64, 4), (64, 5)])
@pytest.mark.parametrize("positions", [300, 200000])
def test_weights_of_long_score_sums(cuda, dtype, tokens, group, positions):
    """A score of 128 dimensions is two sums of 64, added and rounded once. Here the first is 4096 and the second 1.75 units of its
    last place, in four steps of 0.44: the score is off by half a unit (2^-12) at most, where one sum that loses each step would be
    by 1.75. The rest of the tolerance as in test_weights_of_large_scores."""
    c = Case([150, 3], 1, group, 128, 16, "head", dtype, tokens)
    c.q[:] = 1
    key = torch.zeros(128)
    key[:64] = 64
    key[64::16] = 0.4375 * 2.0 ** -11
    for b, n in enumerate(c.lens):
        for p in range(n):
            c.pk[int(c.table[b, p // 16]), :, p % 16] = key.to(dtype).cuda()
    c.kn[:] = key.to(dtype)
    c = with_room(c, positions)
    lse = 512 + 2 * torch.rand(2, tokens, group, generator=torch.Generator().manual_seed(2))
    acc, fresh = (x.cpu().double() for x in kvcache.attention_weights(c.cache, c.q.cuda(), c.kn.cuda(), lse.cuda(), scale=0.125))
    d = 0.125 * (4096 + 1.75 * 2.0 ** -11) - lse.double()
    w = torch.exp(d)
    tol = w * (0.125 * 2.0 ** -12 + 3 * 2.0 ** -24 * d.abs() + 2.0 ** -22 + 2.0 ** -24 * tokens * group)
    for b, n in enumerate(c.lens):
        near(acc[b, 0, :n], w[b].sum().expand(n), tol[b].sum().expand(n), "acc")
        for u in range(tokens):
            near(fresh[b, 0, u:u + 1], w[b, u:].sum()[None], tol[b, u:].sum()[None], "fresh")
