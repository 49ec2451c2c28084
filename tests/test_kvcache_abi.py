"""The paged cache's C entry points refuse bad descriptions before they touch a device (CPU)."""
import ctypes as C

import pytest

from technograd_b200 import _lib

torch = pytest.importorskip("torch")
from technograd_b200 import kvcache  # noqa: E402


def cache(**kw):
    f = dict(type=_lib.BF16, seqs=2, nkv=2, head_dim=64, page=16, pages=8, table_cols=4, max_len=60, k=0x10000, v=0x20000, page_stride=2048,
             head_stride=1024, pos_stride=64, table=0x1000, len=0x2000)
    f.update(kw)
    c = _lib.Kv()
    for n, v in f.items():
        setattr(c, n, v)
    return c


def drafts(**kw):
    f = dict(tokens=3, nq=4, scale=0.1, q=0x30000, q_seq=768, q_tok=256, q_head=64, k=0x40000, v=0x50000, kv_seq=384, kv_tok=128, kv_head=64)
    f.update(kw)
    d = _lib.Drafts()
    for n, v in f.items():
        setattr(d, n, v)
    return d


BAD_CACHE = [dict(type=3), dict(type=-1), dict(seqs=-1), dict(nkv=0), dict(page=0), dict(pages=-1), dict(table_cols=-1), dict(max_len=-1), dict(max_len=65),
             dict(head_dim=0), dict(head_dim=264), dict(head_dim=60), dict(k=0x10008), dict(v=0x20002), dict(page_stride=2044), dict(head_stride=1023),
             dict(pos_stride=-64), dict(k=0), dict(v=0), dict(table=0), dict(len=0), dict(type=_lib.F32, head_dim=66),
             dict(pages=2 ** 31 - 1, page_stride=2 ** 40 + 8), dict(pages=0, table=0)]
BAD_DRAFTS = [dict(tokens=0), dict(tokens=65), dict(nq=0), dict(nq=3), dict(q=0), dict(q=0x30008), dict(q_tok=252), dict(k=0), dict(k=0x40004),
              dict(kv_head=60), dict(kv_tok=-128), dict(q_seq=-768), dict(kv_tok=2 ** 34), dict(q_tok=2 ** 34), dict(nq=2 ** 21)]


def refused(rc):
    assert rc == _lib.EINVAL and _lib.lib().tg_cuda_error()


@pytest.mark.parametrize("c,d", [(cache(**b), drafts()) for b in BAD_CACHE] + [(cache(), drafts(**b)) for b in BAD_DRAFTS])
def test_bad_descriptions(c, d):
    L, p = _lib.lib(), C.byref
    refused(L.tg_cuda_tree_attn_workspace(p(c), p(d)))
    refused(L.tg_cuda_tree_attn(p(c), p(d), 0x60000, 768, 256, 64, 0x70000, None, 0, None))
    refused(L.tg_cuda_attn_weights(p(c), p(d), 0x70000, None, None, 0, 0, 0x80000, 0x90000, None))


@pytest.mark.parametrize("c", [cache(**b) for b in BAD_CACHE])
def test_bad_caches_for_commit_and_evict(c):
    L, p = _lib.lib(), C.byref
    refused(L.tg_cuda_kv_commit(p(c), p(drafts()), None, 0x70000, None, None, 0, 0, 0, None))
    refused(L.tg_cuda_kv_evict(p(c), p(cache()), 0x70000, 120, 60, 32, 4, 1, 0x80000, 0x90000, 0xA0000, None))


def test_other_refusals():
    L, p, c, d = _lib.lib(), C.byref, cache(), drafts()
    out = (0x60000, 768, 256, 64)
    refused(L.tg_cuda_tree_attn(None, p(d), *out, 0x70000, None, 0, None))
    refused(L.tg_cuda_tree_attn(p(c), None, *out, 0x70000, None, 0, None))
    refused(L.tg_cuda_tree_attn(p(c), p(d), None, 768, 256, 64, 0x70000, None, 0, None))
    refused(L.tg_cuda_tree_attn(p(c), p(d), *out, None, None, 0, None))
    refused(L.tg_cuda_tree_attn(p(c), p(d), 0x60008, 768, 256, 64, 0x70000, None, 0, None))
    refused(L.tg_cuda_tree_attn(p(c), p(d), 0x60000, 768, 252, 64, 0x70000, None, 0, None))
    refused(L.tg_cuda_attn_weights(p(c), p(d), None, None, None, 0, 0, 0x80000, 0x90000, None))
    refused(L.tg_cuda_attn_weights(p(c), p(d), 0x70000, None, 0x80000, 128, 64, 0x80000, 0x90000, None))  # in place, other strides
    refused(L.tg_cuda_attn_weights(p(c), p(d), 0x70000, None, None, 0, 0, 0x80000, None, None))
    refused(L.tg_cuda_kv_commit(p(c), p(d), None, None, None, None, 0, 0, 0, None))
    refused(L.tg_cuda_kv_commit(p(c), p(d), None, 0x2000, None, None, 0, 0, 0, None))  # len itself
    refused(L.tg_cuda_kv_commit(p(c), p(d), None, 0x70000, 0x80000, None, 0, 0, 0, None))
    refused(L.tg_cuda_kv_commit(p(c), p(drafts(tokens=0)), None, 0x70000, None, None, 0, 0, 0, None))
    for budget, recent, sink in ((0, 0, 0), (8, 9, 0), (8, 4, 5), (8, -1, 0), (8, 0, -1)):
        refused(L.tg_cuda_kv_evict(p(c), p(c), 0x70000, 120, 60, budget, recent, sink, 0x80000, 0x90000, 0xA0000, None))
    for dst in (cache(type=_lib.F16), cache(nkv=1), cache(head_dim=32), cache(seqs=1)):
        refused(L.tg_cuda_kv_evict(p(c), p(dst), 0x70000, 120, 60, 8, 0, 0, 0x80000, 0x90000, 0xA0000, None))
    refused(L.tg_cuda_kv_evict(p(c), None, 0x70000, 120, 60, 8, 0, 0, 0x80000, 0x90000, 0xA0000, None))
    refused(L.tg_cuda_kv_evict(p(c), p(c), 0x70000, 120, 60, 8, 0, 0, None, 0x90000, 0xA0000, None))


def test_without_a_device_there_is_an_error():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert _lib.lib().tg_cuda_tree_attn_workspace(C.byref(cache()), C.byref(drafts())) < 0


def test_packed_drafts_are_the_structure():
    d = drafts(mask=0x123456789A0, count=0xABCDEF0)
    fields = [getattr(d, n) or 0 for n, _ in _lib.Drafts._fields_]
    assert kvcache._pack_drafts(*fields) == bytes(d)


def test_tensors_on_the_cpu_are_refused():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        kvcache.PagedKV(k, k, torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
