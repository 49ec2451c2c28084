"""Rotary positions and the append to the paged cache: what their C entry points and Python calls refuse (CPU)."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")
from technograd_b200 import _lib, kvcache  # noqa: E402
from test_kvcache_abi import BAD_CACHE, cache, drafts, refused  # noqa: E402
from test_kvcache_host import cache as fake_cache, drafted, library  # noqa: E402, F401

BF16 = torch.bfloat16
OUT = (0x60000, 768, 256, 64)  # q_out
KEYS = (0x70000, 384, 128, 64)  # k_out


def rotary(**kw):
    f = dict(dim=64, interleaved=0, inverse=0, gain=1.0, freq=0x8000, pos=0x9000, pos_seq=3)
    f.update(kw)
    r = _lib.Rotary()
    for n, v in f.items():
        setattr(r, n, v)
    return r


BAD_ROTARY = [dict(dim=-2), dict(dim=66), dict(dim=3), dict(interleaved=2), dict(inverse=-1), dict(freq=0), dict(freq=0x8004), dict(pos=0x9002), dict(pos_seq=-3)]


def rope(r=None, type=_lib.BF16, seqs=2, tokens=3, heads=4, dim=64, x=(0x30000, 768, 256, 64), out=OUT):
    return _lib.lib().tg_cuda_rope(C.byref(rotary() if r is None else r), type, seqs, tokens, heads, dim, *x, *out, None)


def append(c=None, d=None, r=None, q_norm=None, k_norm=None, q=OUT, k=KEYS, lens=0xA0000):
    return _lib.lib().tg_cuda_kv_append(C.byref(cache() if c is None else c), C.byref(drafts() if d is None else d), r if r is None else C.byref(r), q_norm, k_norm,
                                        1e-6, *q, *k, lens, None)


@pytest.mark.parametrize("bad", BAD_ROTARY)
def test_bad_rotations(bad):
    refused(rope(rotary(**bad)))
    refused(append(r=rotary(**bad)))


@pytest.mark.parametrize("bad", [dict(type=3), dict(seqs=-1), dict(tokens=-1), dict(heads=-1), dict(heads=2 ** 21), dict(dim=0), dict(dim=264), dict(dim=60),
                                 dict(type=_lib.F32, dim=66), dict(x=(0, 768, 256, 64)), dict(x=(0x30008, 768, 256, 64)), dict(x=(0x30000, 767, 256, 64)),
                                 dict(x=(0x30000, 768, -256, 64)), dict(out=(0, 768, 256, 64)), dict(out=(0x60004, 768, 256, 64)), dict(out=(0x60000, 768, 256, 60)),
                                 dict(out=(0x60000, 0, 256, 64)), dict(out=(0x60000, 512, 256, 64)), dict(out=(0x60000, 768, 256, -64))])
def test_bad_rows(bad):
    refused(rope(**bad))


def test_in_place_means_the_same_strides():
    """Rows read by one warp would be written by another."""
    refused(rope(out=(0x30000, 384, 128, 64), seqs=2, tokens=3, heads=2))
    refused(rope(out=(0x30000, 768, 64, 192)))
    refused(append(q=(0x30000, 1536, 512, 64)))
    refused(append(k=(0x40000, 384, 64, 192)))


def test_null_rotation():
    refused(_lib.lib().tg_cuda_rope(None, _lib.BF16, 2, 3, 4, 64, 0x30000, 768, 256, 64, *OUT, None))


@pytest.mark.parametrize("c", [cache(**b) for b in BAD_CACHE])
def test_append_refuses_bad_caches(c):
    refused(append(c))


@pytest.mark.parametrize("bad", [dict(tokens=0), dict(nq=0), dict(nq=3), dict(q=0x30008), dict(q_tok=252), dict(k=0), dict(v=0), dict(k=0x40004), dict(kv_head=60),
                                 dict(kv_tok=-128), dict(q_seq=-768), dict(count=0x1002), dict(q=0)])
def test_append_refuses_bad_tokens(bad):
    refused(append(d=drafts(**bad)))  # (without q there is nothing for q_out)


def test_append_refuses_the_rest():
    refused(append(lens=None))
    refused(append(lens=0x2000))  # the cache's own
    refused(append(lens=0xA0002))
    refused(append(q=(None, 768, 256, 64)))
    refused(append(q=(0x60008, 768, 256, 64)))
    refused(append(q=(0x60000, 0, 256, 64)))
    refused(append(k=(0x70008, 384, 128, 64)))
    refused(append(k=(0x70000, 384, 128, 56)))
    refused(append(k=(0x70000, 384, 0, 64)))
    refused(append(q_norm=0x1002))
    refused(append(k_norm=0x1001))
    refused(append(d=drafts(q=0), q=(None, 0, 0, 0), q_norm=0x1000))
    for bad in (dict(head_stride=0), dict(page_stride=1024), dict(pos_stride=56)):  # rows over another would be written in any order
        refused(append(cache(**bad)))
    refused(append(cache(nkv=2 ** 20 + 1, head_stride=0), drafts(q=0), q=(None, 0, 0, 0)))


def test_good_descriptions_get_as_far_as_the_device():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")  # (the addresses are made up)
    for rc in (rope(), rope(out=(0x30000, 768, 256, 64)), rope(rotary(dim=0, freq=0)), rope(rotary(pos=0)), rope(seqs=1, x=(0x30000, 7, 256, 64)),
               append(), append(r=rotary()), append(k=(None, 0, 0, 0)), append(d=drafts(q=0), q=(None, 0, 0, 0)), append(q_norm=0x1000, k_norm=0x1004)):
        assert rc not in (_lib.OK, _lib.EINVAL)


def test_nothing_to_rotate():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for kw in (dict(seqs=0), dict(tokens=0), dict(heads=0)):
        assert rope(x=(0, 0, 0, 0), out=(0, 0, 0, 0), **kw) != _lib.EINVAL


def test_packed_rotation_is_the_structure():
    r = rotary(interleaved=1, inverse=1, gain=1.25, pos_seq=77)
    assert kvcache._pack_rotary(*(getattr(r, n) for n, _ in _lib.Rotary._fields_)) == bytes(r)


def test_frequencies():
    f = kvcache.rotary_frequencies(64, 1e6)
    assert f.dtype is torch.float64 and f.tolist() == pytest.approx([1e6 ** (-i / 32) for i in range(32)], rel=1e-15)
    assert torch.equal(kvcache.rotary_frequencies(64, 1e6, 4.0), f / 4)
    g = kvcache.rotary_frequencies(64, 1e6, 4.0, original=32768)
    turns = 32768 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.allclose(g[turns <= 1], f[turns <= 1] / 4, rtol=1e-15)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and ((g < f) & (g > f / 4))[mid].all() and (g.diff() < 0).all()
    assert kvcache.rotary_frequencies(0).numel() == 0
    for kw in (dict(part=7), dict(part=8, theta=0), dict(part=8, factor=-1.0), dict(part=8, factor=2.0, original=100, fast=1.0)):
        with pytest.raises(ValueError):
            kvcache.rotary_frequencies(**kw)


class Rotation:
    """What the calls read of a Rotary; tensors on the CPU have the device index -1."""
    part, gain, interleaved, index, head_dim, _at = 64, 1.0, False, -1, 64, 0x8000
    _pack = kvcache.Rotary._pack


def test_append_checks_its_arguments(library):  # noqa: F811
    q, k, v = drafted()
    r, pos, norm = Rotation(), torch.zeros(2, 3, dtype=torch.int32), torch.ones(64)
    good = dict(cache=fake_cache(), k=k, v=v, q=q, rotary=r, pos=pos, q_norm=norm, k_norm=norm)
    for bad in (dict(pos=pos.long()), dict(pos=pos[:1]), dict(pos=pos[:, :2]), dict(pos=torch.zeros(3, 2, dtype=torch.int32).t()), dict(q=None), dict(q_norm=norm[:32]),
                dict(k_norm=norm.double()), dict(rotary=None), dict(count=torch.zeros(2)), dict(v=v[:, :2]), dict(q=q[:, :2]), dict(cache=fake_cache(head_dim=32))):
        with pytest.raises(ValueError):
            kvcache.append(**{**good, **bad})
    other = Rotation()
    other.head_dim = 32
    with pytest.raises(ValueError):
        kvcache.append(**{**good, "rotary": other})
    assert not library.calls
    for kw in (dict(), dict(pos=None), dict(pos=pos[0]), dict(pos=pos[:1].expand(2, 3)), dict(keys=True), dict(rotary=None, pos=None), dict(q=None, q_norm=None)):
        lens, qr, kr = kvcache.append(**{**good, **kw})
        assert (qr is None) == (kw.get("q", q) is None) and (kr is not None) == ("keys" in kw) and lens.shape == (2,)
    assert [n for n, _ in library.calls] == ["tg_cuda_kv_append"] * 7


def test_a_gradient_through_append_is_an_error(library):  # noqa: F811
    for which in range(3):
        q, k, v = (x.requires_grad_(i == which) for i, x in enumerate(drafted()))
        _, qr, kr = kvcache.append(fake_cache(), k, v, q=q, keys=True)
        for y in (qr, kr):
            with pytest.raises(RuntimeError, match="append has no backward"):
                y.float().sum().backward(retain_graph=True)
        with torch.no_grad():
            assert not any(y.requires_grad for y in kvcache.append(fake_cache(), k, v, q=q, keys=True))


def test_tensors_on_the_cpu_are_refused():
    with pytest.raises(ValueError):
        kvcache.Rotary(64, freq=torch.ones(32, dtype=torch.float64))
    with pytest.raises(ValueError):
        kvcache.rope(torch.zeros(1, 1, 1, 64), Rotation())
