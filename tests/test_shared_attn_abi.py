"""Attention below shared prefixes: what its C entry points and its Python calls refuse (CPU)."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
from technograd_b200 import _lib, kvcache  # noqa: E402
from test_kvcache_abi import BAD_CACHE, BAD_DRAFTS, cache, drafts, refused  # noqa: E402
from test_kvcache_host import cache as fake_cache, drafted, library  # noqa: E402, F401

OUT = (0x60000, 768, 256, 64)


def prefix(**kw):
    f = dict(groups=1, max_shared=32, max_own=28, first=0x8000, members=0x8100, shared=0x8200, group=0x8300)
    f.update(kw)
    x = _lib.Prefix()
    for n, v in f.items():
        setattr(x, n, v)
    return x


def size(c=None, d=None, x=None):
    return _lib.lib().tg_cuda_shared_attn_workspace(C.byref(c or cache()), C.byref(d or drafts()), C.byref(x or prefix()))


def attend(c=None, d=None, x=None, out=OUT, lse=0x70000, work=0x90000, n=1 << 30):
    return _lib.lib().tg_cuda_shared_attn(C.byref(c or cache()), C.byref(d or drafts()), C.byref(x or prefix()), *out, lse, work, n, None)


@pytest.mark.parametrize("bad", BAD_CACHE)
def test_bad_caches(bad):
    refused(size(cache(**bad)))
    refused(attend(cache(**bad)))


@pytest.mark.parametrize("bad", BAD_DRAFTS)
def test_bad_drafts(bad):
    refused(size(d=drafts(**bad)))
    refused(attend(d=drafts(**bad)))


@pytest.mark.parametrize("bad", [dict(groups=-1), dict(groups=3), dict(max_shared=-1), dict(max_shared=61), dict(max_own=-1), dict(first=0), dict(members=0), dict(shared=0),
                                 dict(group=0), dict(first=0x8002), dict(members=0x8101), dict(shared=0x8203), dict(group=0x8302), dict(always=2), dict(always=-1)])
def test_bad_prefixes(bad):
    refused(size(x=prefix(**bad)))
    refused(attend(x=prefix(**bad)))


@pytest.mark.parametrize("bad", [dict(out=(0, 768, 256, 64)), dict(out=(0x60008, 768, 256, 64)), dict(out=(0x60000, 768, 252, 64)), dict(out=(0x60000, 0, 256, 64)),
                                 dict(out=(0x60000, 512, 256, 64)), dict(out=(0x60000, 768, 256, -64)), dict(lse=None), dict(lse=0x70002)])
@pytest.mark.parametrize("kw", [dict(groups=0), dict(always=0), dict(always=1)])
def test_bad_outputs(bad, kw):
    refused(attend(x=prefix(**kw), **bad))


def test_null():
    L, p = _lib.lib(), C.byref
    for c, d, x in ((None, drafts(), prefix()), (cache(), None, prefix()), (cache(), drafts(), None)):
        a = [None if y is None else p(y) for y in (c, d, x)]
        refused(L.tg_cuda_shared_attn_workspace(*a))
        refused(L.tg_cuda_shared_attn(*a, *OUT, 0x70000, None, 0, None))


def test_good_descriptions_get_as_far_as_the_device():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")  # (the addresses are made up)
    for x in (prefix(), prefix(max_own=10 ** 9), prefix(groups=0, first=0, members=0, shared=0, group=0), prefix(max_shared=0)):
        assert size(x=x) < 0 and size(x=x) != _lib.EINVAL
        assert attend(x=x) not in (_lib.OK, _lib.EINVAL)


def fake(**kw):
    return fake_cache(device=torch.device("cpu"), table=torch.zeros(kw.get("seqs", 2), 4, dtype=torch.int32), **kw)


def test_groups_are_checked():
    c = fake(seqs=6)
    for bad in ([(0, 7, 16)], [(-1, 2, 16)], [(0, 2, 16), (1, 2, 16)], [(2, 2, 16), (0, 2, 16)], [(0, 0, 16)], [(0, 2, -1)], [(0, 2, 65)]):
        with pytest.raises(ValueError):
            kvcache.SharedPrefix(c, bad)
    with pytest.raises(ValueError):
        kvcache.SharedPrefix(c, [], max_own=-1)
    with pytest.raises(ValueError, match="32 bits"):
        kvcache.SharedPrefix(c, [], max_own=2 ** 32)
    x = kvcache.SharedPrefix(c, [(0, 2, 16), (3, 3, 32)])
    s = x._struct
    assert (s.groups, s.max_shared, s.max_own) == (2, 32, 40)  # sequence 2 shares nothing
    assert x._held.tolist() == [0, 3, 2, 3, 16, 32, 0, 0, -1, 1, 1, 1]
    assert [s.members - s.first, s.shared - s.first, s.group - s.first] == [8, 16, 24]
    assert kvcache.SharedPrefix(c, [(0, 6, 16)])._struct.max_own == 24 and kvcache.SharedPrefix(c, [])._struct.groups == 0


def test_attention_checks_its_arguments(library):  # noqa: F811
    c, (q, k, v) = fake(), drafted()
    x = kvcache.SharedPrefix(c, [(0, 2, 16)])
    for kw in (dict(cache=fake(seqs=3)), dict(cache=fake(max_len=15)), dict(q=q[:, :2]), dict(v=v[:1]), dict(k=k.float()), dict(mask=torch.zeros(2, 3)), dict(count=torch.zeros(2))):
        with pytest.raises(ValueError):
            kvcache.shared_attention(**{**dict(cache=c, prefix=x, q=q, k=k, v=v), **kw})
    assert not library.calls
    out, lse = kvcache.shared_attention(c, x, q, k, v)
    assert out.shape == q.shape and lse.shape == q.shape[:3]
    assert [n for n, _ in library.calls] == ["tg_cuda_shared_attn_workspace", "tg_cuda_shared_attn"]


def test_scratch_lives_until_the_call_returns(library):  # noqa: F811
    import gc
    held = []

    def look(name, args):
        if name == "tg_cuda_shared_attn":
            work, n = args[8], args[9]
            held.append(any(type(y) is torch.Tensor and y.data_ptr() <= work and work + n <= y.data_ptr() + y.nbytes for y in gc.get_objects()))
    library.on_call = look
    c = fake()
    x = kvcache.SharedPrefix(c, [(0, 2, 16)])
    for _ in range(2):  # the plan made, and the plan found
        kvcache.shared_attention(c, x, *drafted())
    assert held == [True, True]


def test_a_gradient_is_an_error(library):  # noqa: F811
    c = fake()
    x = kvcache.SharedPrefix(c, [(0, 2, 16)])
    for which in range(3):
        args = [y.requires_grad_(i == which) for i, y in enumerate(drafted())]
        for y in kvcache.shared_attention(c, x, *args):
            with pytest.raises(RuntimeError, match="shared_attention has no backward"):
                y.float().sum().backward(retain_graph=True)
    assert not any(y.requires_grad for y in kvcache.shared_attention(c, x, *drafted()))
