"""The paged cache's Python calls, up to the library's entry points: a stand-in takes the place of the library (CPU)."""
import gc
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")
from technograd_b200 import kvcache  # noqa: E402

BF16 = torch.bfloat16


def cache(**kw):
    """What the calls read of a PagedKV; tensors on the CPU have the device index -1."""
    f = dict(index=-1, dtype=BF16, seqs=2, nkv=2, head_dim=64, page=16, scale=0.125, max_len=40, lens=torch.zeros(2, dtype=torch.int32),
             _at=0, _plans={}, _one=torch.empty(1))
    return SimpleNamespace(**{**f, **kw})


def drafted(seqs=2, tokens=3, nq=4, nkv=2, dim=64):
    return tuple(torch.zeros(seqs, tokens, h, dim, dtype=BF16) for h in (nq, nkv, nkv))


@pytest.fixture
def library(monkeypatch):
    """A library whose entry points succeed and leave their arguments in `calls`."""
    class Library:
        size, calls, on_call = 4096, [], None

        def __getattr__(self, name):
            def call(*args):
                self.calls.append((name, args))
                if self.on_call:
                    self.on_call(name, args)
                return self.size if name.endswith("_workspace") else 0
            return call
    L = Library()
    L.calls = []
    monkeypatch.setattr(kvcache._lib, "lib", lambda: L)
    monkeypatch.setattr(kvcache._lib, "check", lambda rc: None)
    monkeypatch.setattr(kvcache, "_stream", lambda c: 0)
    return L


def test_scratch_lives_until_the_call_returns(library):
    """Once no tensor holds it, its memory may be anybody's before the kernels that use it are launched."""
    held = []

    def look(name, args):
        if name == "tg_cuda_tree_attn":
            work, size = args[7], args[8]
            held.append(any(type(x) is torch.Tensor and x.data_ptr() <= work and work + size <= x.data_ptr() + x.nbytes for x in gc.get_objects()))
    library.on_call = look
    c = cache()
    for _ in range(2):  # the plan made, and the plan found
        kvcache.tree_attention(c, *drafted())
    assert held == [True, True]
