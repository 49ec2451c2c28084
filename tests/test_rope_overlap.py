"""Rotations and appends whose outputs lie over what the call reads: one warp would read what another has written (CPU)."""
import ctypes as C
import itertools
import random

import pytest

torch = pytest.importorskip("torch")
from technograd_b200 import _lib  # noqa: E402
from test_kvcache_abi import cache, drafts, refused  # noqa: E402
from test_rope_abi import append, rope, rotary  # noqa: E402

X, ROW, DIM = 0x30000, 64 * 2, 64


def accepted(rc):
    return rc not in (_lib.OK, _lib.EINVAL)  # past the checks only the device is missing


@pytest.fixture
def no_gpu():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")  # (the addresses are made up)


@pytest.mark.parametrize("shift", [ROW, -ROW, 3 * ROW, 16, -16, 4 * ROW, 12 * ROW, 24 * ROW - ROW])
def test_shifted_outputs(shift):
    """x[:, :, 0:4] into x[:, :, 1:5] and the like, by heads, tokens, sequences and parts of a row."""
    refused(rope(x=(X, 768, 256, 64), out=(X + shift, 768, 256, 64)))


def test_heads_beside_each_other(no_gpu):
    """Disjoint heads of one projection's rows lie between each other."""
    x = dict(seqs=2, tokens=3, heads=4)
    for first, ok in ((0, True), (3, False), (4, False), (7, False), (8, True), (10, True)):  # x has heads 4 to 7 of 14
        got = rope(x=(X + 4 * ROW, 3 * 14 * 64, 14 * 64, 64), out=(X + first * ROW, 3 * 14 * 64, 14 * 64, 64), **x)
        assert (accepted(got) if ok or first == 4 else got == _lib.EINVAL), first
    assert accepted(rope(x=(X, 768, 256, 64), out=(X + 24 * ROW, 768, 256, 64)))
    assert accepted(rope(x=(X + 24 * ROW, 768, 256, 64), out=(X, 768, 256, 64)))


def places(at, strides, n):
    return {(at + 2 * sum(s * i for s, i in zip(strides, index))) // 16 + piece for index in itertools.product(*map(range, n)) for piece in range(8)}


def test_against_all_rows(no_gpu):
    """Layouts of the same strides to the row; of others, what shares memory is never accepted."""
    r, met = random.Random(5), [0, 0]
    for _ in range(3000):
        n = [r.randint(1, 4) for _ in range(3)]

        def layout():
            strides, span = [0] * 3, 64
            for i in r.sample(range(3), 3):
                strides[i] = span + 8 * r.randint(0, 3) * r.randint(0, 30)
                span = strides[i] * n[i] if r.random() < 0.5 else strides[i] * (n[i] - 1) + span
            return strides
        a = layout()
        b = a if r.random() < 0.7 else layout()
        shift = r.randint(-40, 40) * 16 if r.random() < 0.5 else r.randint(-4000, 4000) * 16
        if shift == 0:
            continue
        meet = not places(X * 16, a, n).isdisjoint(places(X * 16 + shift, b, n))
        got = rope(rotary(pos=0), seqs=n[0], tokens=n[1], heads=n[2], x=(X * 16, *a), out=(X * 16 + shift, *b))
        if meet:
            assert got == _lib.EINVAL, (n, a, b, shift)
        elif a == b:
            assert accepted(got), (n, a, b, shift)
        met[meet] += 1
    assert min(met) > 300


def test_expanded_input(no_gpu):
    """One row for all tokens and heads: not to be written while it is read."""
    one = (X, 0, 0, 0)
    assert accepted(rope(x=one, out=(X + ROW, 768, 256, 64))) and accepted(rope(x=one, out=(X - 24 * ROW, 768, 256, 64)))
    refused(rope(x=(X + 5 * ROW, 0, 0, 0), out=(X, 768, 256, 64)))


def test_append_outputs_over_other_inputs():
    """q_out and k_out may be q and k; over v, each other's input or each other they are refused."""
    q, k, v = (0x30000, 768, 256, 64), (0x40000, 384, 128, 64), (0x50000, 384, 128, 64)
    for kw in (dict(k=v), dict(q=(0x50000, 768, 256, 64)), dict(q=(0x40000, 768, 256, 64)), dict(k=(0x30000, 384, 128, 64)), dict(k=(0x30000 + 5 * ROW, 384, 128, 64)),
               dict(q=(0x30000 + ROW, 768, 256, 64)), dict(k=(0x40000 - ROW, 384, 128, 64)), dict(q=(0x60000, 768, 256, 64), k=(0x60000 + 2 * ROW, 384, 128, 64))):
        refused(append(**kw))
    if not torch.cuda.is_available():
        for kw in (dict(q=q, k=k), dict(q=q), dict(k=k)):
            assert accepted(append(**kw))


def test_append_of_a_projection_in_place(no_gpu):
    """q, k and v of one projection's rows [2][3][4 + 2 + 2][64], rotated where they are; and into the columns of another's."""
    s = (3 * 8 * 64, 8 * 64, 64)
    d = drafts(q=X, q_seq=s[0], q_tok=s[1], k=X + 4 * ROW, v=X + 6 * ROW, kv_seq=s[0], kv_tok=s[1])
    assert accepted(append(d=d, q=(X, *s), k=(X + 4 * ROW, *s)))
    assert accepted(append(d=d, q=(0x60000, *s), k=(0x60000 + 4 * ROW, *s)))
    for q, k in ((0, 6), (2, 4), (0, 3), (4, 0)):
        assert append(d=d, q=(X + q * ROW, *s), k=(X + k * ROW, *s)) == _lib.EINVAL


@pytest.mark.parametrize("at", [0x2000, 0x2004, 0x1ffc, 0x7000, 0x7004])
def test_new_lengths_over_what_is_read(at):
    """Of 2 sequences' len at 0x2000 and count at 0x7000."""
    d = drafts(count=0x7000)
    refused(append(d=d, lens=at))
    refused(_lib.lib().tg_cuda_kv_commit(C.byref(cache()), C.byref(d), None, at, None, None, 0, 0, 0, None))


@pytest.mark.parametrize("at", [0x2008, 0x1ff8, 0x7008])
def test_new_lengths_beside_what_is_read(no_gpu, at):
    assert accepted(append(d=drafts(count=0x7000), lens=at))
    assert accepted(_lib.lib().tg_cuda_kv_commit(C.byref(cache()), C.byref(drafts(count=0x7000)), None, at, None, None, 0, 0, 0, None))
