"""Angles of rotations against integers (GPU): pos freq / 2 pi, freq being the given f64 and 1 / 2 pi having 300 bits.

The header's bounds: the angle to 2^-29, cos and sin of it to 2^-23. Rows (1, 0) turn into (cos, sin), with no further rounding in f32."""
import math

import pytest
import torch

from technograd_b200 import kvcache
from test_gpu_kvcache import F32, Case, reported

pytestmark = pytest.mark.gpu
BITS = 300


def arctan(n):
    """2^BITS arctan(1 / n)."""
    total, term, k = 0, (1 << BITS) // n, 1
    while term:
        total += (term // k) * (1 if k % 4 == 1 else -1)
        term, k = term // (n * n), k + 2
    return total


TWO_PI = 8 * (4 * arctan(5) - arctan(239))  # 2^BITS times it, but for a few units
ONE_TURN = (1 << 2 * BITS) // TWO_PI  # 2^BITS / 2 pi


def angles(pos, freq):
    """pos freq but for whole turns, [positions][frequencies] f64."""
    def one(p, f):
        m, d = f.as_integer_ratio()
        turns = m * p * ONE_TURN // d % (1 << BITS)
        turns -= (turns >> BITS - 1) << BITS
        return (turns * TWO_PI >> BITS) / (1 << BITS)
    return torch.tensor([[one(p, f) for f in freq] for p in pos], dtype=torch.float64)


def check(got, want, what):
    """got [rows][2 half] of rows (1, 0), f32, want their angles."""
    half = want.shape[1]
    for x, y in ((got[:, :half].double().cpu(), want.cos()), (got[:, half:].double().cpu(), want.sin())):
        assert (x - y).abs().max() <= 2.0 ** -23 + 2.0 ** -29, (what, float((x - y).abs().max()))


def test_two_pi():
    assert abs(TWO_PI / (1 << BITS) - 2 * math.pi) < 1e-15


FREQUENCIES = [kvcache.rotary_frequencies(256, 1e4), kvcache.rotary_frequencies(256, 1e6, 4.0, 32768), kvcache.rotary_frequencies(256, 5e5, 8.0),
               torch.tensor([(-1) ** i * 3.7 ** (i / 4 - 20) for i in range(128)], dtype=torch.float64)]  # 1e-12 to 1e6, of both signs


@pytest.mark.parametrize("freq", FREQUENCIES)
@pytest.mark.parametrize("inverse", [False, True])
def test_angles(cuda, freq, inverse):
    """Near positions, far ones, and those at the ends of 32 bits."""
    g = torch.Generator().manual_seed(30)
    pos = torch.cat([torch.randint(-top, top, (40,), generator=g) for top in (100, 1 << 14, 1 << 20, 1 << 24, 1 << 27, 1 << 31)] +
                    [torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 24 + 1, 2 ** 30 + 1])]).to(torch.int32)
    x = torch.zeros(1, len(pos), 1, 256, device="cuda")
    x[..., :128] = 1
    y = kvcache.rope(x, kvcache.Rotary(256, freq.cuda()), pos.cuda(), inverse)
    check(y[0, :, 0], angles([-p if inverse else p for p in pos.tolist()], freq.tolist()), "y")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("part,pairs", [(16, False), (16, True), (14, False)])
@pytest.mark.parametrize("inverse", [False, True])
def test_frequencies_that_are_no_numbers(cuda, dtype, part, pairs, inverse):
    """NaN, at position 0 too, as the formula has it (0 times infinity), in that pair alone."""
    freq = [1.0, math.nan, 0.5, math.inf, -math.inf, 0.0, 1e-300, 1e300][:part // 2]
    x = torch.randn(1, 3, 5, 16, generator=torch.Generator().manual_seed(31)).to(dtype).cuda()
    y = kvcache.rope(x, kvcache.Rotary(16, torch.tensor(freq, dtype=torch.float64).cuda(), interleaved=pairs), torch.tensor([0, 1, 7], dtype=torch.int32, device="cuda"), inverse)
    bad = torch.zeros(16, dtype=torch.bool)
    for i, f in enumerate(freq):
        if not math.isfinite(f):
            for e in (2 * i, 2 * i + 1) if pairs else (i, i + part // 2):
                bad[e] = True
    assert torch.isnan(y[..., bad.cuda()]).all() and torch.isfinite(y[..., ~bad.cuda()]).all()


@pytest.mark.parametrize("part", [16, 6])
def test_positions_behind_a_cache_of_nearly_32_bits(cuda, part):
    """len + i past 2^31: such a row is not written to the cache, and its angle is that of its own position."""
    dim, T, top = 16, 70000, 0x7fff0000
    k = torch.zeros(0, 1, 1 << 30, dim, device="cuda")
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    r = kvcache.Rotary(dim, theta=1e4, part=part)
    cache = kvcache.PagedKV(k, k, table, torch.tensor([top - 7], dtype=torch.int32, device="cuda"), max_len=top)
    x = torch.zeros(1, T, 1, dim, device="cuda")
    x[..., :part // 2] = 1
    lens, q, kr = kvcache.append(cache, x, x, q=x, rotary=r, keys=True)
    good = Case([5], 1, 1, 64, 16, "head", F32, 1)
    assert "past the table" in reported(lambda: kvcache.tree_attention(good.cache, good.q.cuda(), good.kn.cuda(), good.vn.cuda()))
    assert lens.tolist() == [2 ** 31 - 1]
    at = [0, 1, 65535, 65536 + 6, 65536 + 7, 65536 + 8, T - 1]
    want = angles([top - 7 + i for i in at], r.freq.tolist())
    check(q[0, at, 0, :part], want, "q"), check(kr[0, at, 0, :part], want, "k")
