"""The paged cache's Python calls, up to the library's entry points: a stand-in takes the place of the library (CPU)."""
import ctypes as C
import gc
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")
from technograd_b200 import kvcache  # noqa: E402
from test_kvcache_abi import cache as kv, drafts  # noqa: E402

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


def test_strides_of_single_rows_do_not_matter(library):
    """k and v of one token, head or sequence are the same rows whatever their strides along it."""
    c = cache(seqs=1)
    q, k, v = drafted(1, 1)
    qkv = torch.zeros(1, 5, 8 * 64, dtype=BF16)[:, 2:3].unflatten(2, (8, 64))
    assert qkv[:, :, 6:].stride() != k.stride()
    kvcache.tree_attention(c, q, k, qkv[:, :, 6:])
    kvcache.commit(c, k, qkv[:, :, 6:], torch.zeros(1, dtype=torch.int32))
    assert [n for n, _ in library.calls[-2:]] == ["tg_cuda_tree_attn", "tg_cuda_kv_commit"]


def test_strides_of_several_rows_do(library):
    c = cache()
    q, k, v = drafted()
    with pytest.raises(ValueError):
        kvcache.tree_attention(c, q, k, v.transpose(1, 2).contiguous().transpose(1, 2))
    assert not library.calls


def test_the_library_does_not_look_at_strides_of_single_rows():
    """A stride along one element alone may be anything: past the checks only the device is missing here."""
    L, p = kvcache._lib.lib(), C.byref
    one = dict(seqs=1, nkv=1, pages=1, page=64, table_cols=1)
    for c, d in ((kv(**one, page_stride=7, head_stride=1), drafts(tokens=1, nq=1, q_seq=1, q_tok=3, q_head=-1, kv_seq=5, kv_tok=1, kv_head=1)),
                 (kv(page=1, pages=64, table_cols=64, pos_stride=-1), drafts())):
        assert L.tg_cuda_tree_attn_workspace(p(c), p(d)) != kvcache._lib.EINVAL
    for c, d in ((kv(page_stride=7), drafts()), (kv(head_stride=1), drafts()), (kv(), drafts(q_seq=1)), (kv(), drafts(kv_tok=1)), (kv(), drafts(kv_head=-8))):
        assert L.tg_cuda_tree_attn_workspace(p(c), p(d)) == kvcache._lib.EINVAL


@pytest.mark.parametrize("seq,head,cols,good", [(200, 100, 100, True), (100, 900, 100, True), (250, 120, 100, True), (200, 100, 101, False), (0, 100, 100, False),
                                                (200, 0, 100, False), (100, 100, 100, False), (150, 100, 100, False), (100, 850, 100, False), (-200, 100, 100, False)])
def test_commit_refuses_weights_whose_rows_overlap(seq, head, cols, good):
    """Several warps would write one element. The description is one that no launch takes (too many tokens), since its addresses
    are made up: past the checks only the device is missing here."""
    if good and torch.cuda.is_available():
        pytest.skip("a GPU is present")
    rc = kvcache._lib.lib().tg_cuda_kv_commit(C.byref(kv(seqs=9)), C.byref(drafts(tokens=2 ** 31 - 1)), None, 0x70000, 0x80000, 0x90000, seq, head, cols, None)
    assert (rc != kvcache._lib.EINVAL) == good


@pytest.mark.parametrize("bad", [dict(head_stride=0), dict(pos_stride=0), dict(page_stride=0), dict(page_stride=1024), dict(head_stride=64), dict(pos_stride=56)])
def test_pools_whose_rows_overlap_are_not_written(bad):
    """A broadcast pool may be read, but a commit or an eviction would write its rows in any order."""
    L, p, c = kvcache._lib.lib(), C.byref, kv(**bad)
    assert L.tg_cuda_kv_commit(p(c), p(drafts()), None, 0x70000, None, None, 0, 0, 0, None) == kvcache._lib.EINVAL
    assert L.tg_cuda_kv_evict(p(kv()), p(c), 0x70000, 120, 60, 32, 4, 1, 0x80000, 0x90000, 0xA0000, None) == kvcache._lib.EINVAL
    assert L.tg_cuda_tree_attn_workspace(p(c), p(drafts())) != kvcache._lib.EINVAL


@pytest.mark.parametrize("out", [(0, 256, 64), (768, 0, 64), (768, 256, 0), (512, 256, 64), (768, 192, 64), (768, 256, 56), (-768, 256, 64)])
def test_outputs_whose_rows_overlap_are_refused(out):
    L, p = kvcache._lib.lib(), C.byref
    assert L.tg_cuda_tree_attn(p(kv()), p(drafts()), 0x60000, *out, 0x70000, None, 0, None) == kvcache._lib.EINVAL


@pytest.mark.parametrize("which", [0, 1, 2])
def test_a_gradient_through_attention_is_an_error(library, which):
    """... and not left out in silence; without autograd, and for inputs that want none, results are plain tensors."""
    x = [y.requires_grad_(i == which) for i, y in enumerate(drafted())]
    out, lse = kvcache.tree_attention(cache(), *x)
    for y in (out, lse):
        with pytest.raises(RuntimeError, match="no backward"):
            (y.float().sum() + x[which].float().sum()).backward(retain_graph=True)
    with torch.no_grad():
        assert not any(y.requires_grad for y in kvcache.tree_attention(cache(), *x))
    assert not any(y.requires_grad for y in kvcache.tree_attention(cache(), *drafted()))


def test_numbers_past_32_bits_are_refused(library):
    """ctypes would pass on their low bits: a budget of 2^32 + 8 as 8."""
    acc = torch.zeros(2, 2, 40)
    for kw in (dict(budget=2 ** 32 + 8), dict(budget=8, recent=2 ** 32), dict(budget=8, sink=2 ** 32 + 1), dict(budget=8, recent=-2 ** 32)):
        with pytest.raises(ValueError, match="32 bits"):
            kvcache.evict(cache(), cache(), acc, **kw)
    assert not library.calls
    kvcache.evict(cache(), cache(), acc, 8, 2, 1)
    assert library.calls[-1][0] == "tg_cuda_kv_evict"


def test_pointers_off_their_type_are_refused():
    """A kernel that reads a word across its boundary would fault."""
    L, p = kvcache._lib.lib(), C.byref
    E = kvcache._lib.EINVAL
    out = (0x60000, 768, 256, 64)
    for c, d in ((kv(table=0x1002), drafts()), (kv(len=0x2001), drafts()), (kv(), drafts(mask=0x3004)), (kv(), drafts(count=0x3002))):
        assert L.tg_cuda_tree_attn_workspace(p(c), p(d)) == E
        assert L.tg_cuda_tree_attn(p(c), p(d), *out, 0x70000, None, 0, None) == E
        assert L.tg_cuda_attn_weights(p(c), p(d), 0x70000, None, None, 0, 0, 0x80000, 0x90000, None) == E
        assert L.tg_cuda_kv_commit(p(c), p(d), None, 0x70000, None, None, 0, 0, 0, None) == E
    c, d = kv(), drafts()
    assert L.tg_cuda_tree_attn(p(c), p(d), *out, 0x70002, None, 0, None) == E
    for at in range(5):
        w = [0x70000, 0xA0000, 0xB0000, 0x80000, 0x90000]  # lse, select, acc, acc_out, fresh
        w[at] += 4 if at == 1 else 2
        assert L.tg_cuda_attn_weights(p(c), p(d), w[0], w[1], w[2], 128, 64, w[3], w[4], None) == E
    for at in range(4):
        w = [0x70000, 0x80000, 0x90000, 0xA0000]  # path, len_out, fresh, acc; and acc, keep, acc_out, len_out
        w[at] += 1
        assert L.tg_cuda_kv_commit(p(c), p(d), w[0], w[1], w[2], w[3], 200, 100, 100, None) == E
        assert L.tg_cuda_kv_evict(p(kv()), p(c), w[0], 120, 60, 32, 4, 1, w[1], w[2], w[3], None) == E


@pytest.mark.parametrize("seq,head", [(-120, 60), (120, -60)])
def test_negative_strides_of_weights_are_refused(seq, head):
    L, p, E = kvcache._lib.lib(), C.byref, kvcache._lib.EINVAL
    assert L.tg_cuda_attn_weights(p(kv()), p(drafts()), 0x70000, None, 0xB0000, seq, head, 0x80000, 0x90000, None) == E
    assert L.tg_cuda_kv_evict(p(kv()), p(kv()), 0xB0000, seq, head, 32, 4, 1, 0x80000, 0x90000, 0xA0000, None) == E
