"""A decoder's key/value cache in pages, over libtgcuda: attention of drafted tokens, the attention
weight each position receives, the commit of accepted tokens, and eviction by that weight.

The pools are torch CUDA tensors [pages, nkv, page, head_dim] (any strides, rows contiguous) in f32,
f16 or bf16; position p of sequence b is row p % page of page table[b, p // page]. Everything is
asynchronous on the current stream; results are new tensors, except that `commit` writes the cache's
pages (and `acc`) and `evict` the destination's. No reference counterpart: the reference recomputes
every position's keys and values (examples/qwen3/import.py:90-132).

A speculative decode step: draft tokens and their mask, `tree_attention` in every layer, compare
with the model's own choices, `commit` the accepted path. When the cache is full, `evict` by the
weights that `attention_weights` has summed up (examples/speculative.py runs all of it)."""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib

_TYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _tensor(name: str, x, dtype, shape, device, contiguous: bool = True) -> None:
    """x is a tensor of this type, shape (None = any extent) and device."""
    if x.dtype is not dtype or x.device != device or len(x.shape) != len(shape) or \
            any(w is not None and w != n for w, n in zip(shape, x.shape)) or (contiguous and not x.is_contiguous()):
        raise ValueError(f"{name}: expected {'a contiguous' if contiguous else 'a'} {dtype} tensor {tuple(shape)} on {device}, got "
                         f"{x.dtype} {tuple(x.shape)} strides {x.stride()} on {x.device}")


def _stream(device) -> int:
    _need(device.index == torch.cuda.current_device(), f"the tensors are on {device}, which is not the current device")
    return torch.cuda.current_stream().cuda_stream


class PagedKV:
    """One layer's cache: pools k and v, the table of pages [seqs, cols] and lengths [seqs] (int32).

    max_len bounds every entry of lens (default: what the table holds); it sizes the launches, so a
    bound near the longest sequence is best."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, max_len: int | None = None):
        _need(k.dim() == 4 and k.dtype in _TYPES and k.is_cuda, "k: expected an f32, f16 or bf16 CUDA tensor [pages, nkv, page, head_dim]")
        _need(k.shape[3] <= 1 or k.stride(3) == 1, "k: the head dimension must be contiguous")
        _need(v.dtype is k.dtype and v.device == k.device and v.shape == k.shape and v.stride() == k.stride(),
              "v: expected k's type, device, shape and strides")
        _tensor("table", table, torch.int32, (None, None), k.device)
        _tensor("lens", lens, torch.int32, (table.shape[0],), k.device)
        self.k, self.v, self.table, self.lens = k, v, table, lens
        self.device, self.dtype = k.device, k.dtype
        self.seqs, cols = table.shape
        pages, self.nkv, self.page, self.head_dim = k.shape
        self.max_len = self.page * cols if max_len is None else int(max_len)
        s = _lib.Kv(_TYPES[k.dtype], self.seqs, self.nkv, self.head_dim, self.page, pages, cols, self.max_len,
                    k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), table.data_ptr(), lens.data_ptr())
        self._struct = s
        self._at = C.addressof(s)

    def with_lens(self, lens: torch.Tensor, max_len: int | None = None) -> "PagedKV":
        """The same pages with other lengths (what `commit` returned)."""
        return PagedKV(self.k, self.v, self.table, lens, max_len)


def _drafts(cache: PagedKV, q, k, v, mask, count, scale):
    B, T = k.shape[0], k.shape[1]
    nkv, dim, dt, dev = cache.nkv, cache.head_dim, cache.dtype, cache.device
    _tensor("k", k, dt, (cache.seqs, None, nkv, dim), dev, False)
    kb, kt, kh, kd = k.stride()
    _need(kd == 1 or dim == 1, "k: the head dimension must be contiguous")
    d = _lib.Drafts()
    d.tokens, d.k, d.kv_seq, d.kv_tok, d.kv_head = T, k.data_ptr(), kb, kt, kh
    if v is not None:
        _tensor("v", v, dt, k.shape, dev, False)
        _need(v.stride() == (kb, kt, kh, kd), "v: expected k's strides")
        d.v = v.data_ptr()
    if q is not None:
        _tensor("q", q, dt, (B, T, None, dim), dev, False)
        d.nq, d.q = q.shape[2], q.data_ptr()
        d.q_seq, d.q_tok, d.q_head, qd = q.stride()
        _need(qd == 1 or dim == 1, "q: the head dimension must be contiguous")
    if mask is not None:
        _tensor("mask", mask, torch.int64, (B, T), dev)
        d.mask = mask.data_ptr()
    if count is not None:
        _tensor("count", count, torch.int32, (B,), dev)
        d.count = count.data_ptr()
    d.scale = 1 / math.sqrt(dim) if scale is None else scale
    return d


def tree_attention(cache: PagedKV, q, k, v, mask=None, count=None, scale: float | None = None):
    """Attention of drafted tokens over the cache and each other (tg_cuda_tree_attn).

    q [seqs, tokens, nq, head_dim]; k, v [seqs, tokens, nkv, head_dim], not yet in the cache; at most 64
    tokens. mask int64 [seqs, tokens]: bit u of an entry = the token attends to drafted token u (None:
    a chain). count int32 [seqs]: tokens drafted (None: all). Returns (out as q, lse f32 [seqs, tokens,
    nq]); a token that sees nothing has out 0 and lse -inf."""
    d = _drafts(cache, q, k, v, mask, count, scale)
    stream, L = _stream(cache.device), _lib.lib()
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
    at = C.byref(d)
    size = L.tg_cuda_tree_attn_workspace(cache._at, at)
    if size < 0:
        _lib.check(size)
    work = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    ob, ot, oh, _ = out.stride()
    _lib.check(L.tg_cuda_tree_attn(cache._at, at, out.data_ptr(), ob, ot, oh, lse.data_ptr(), work.data_ptr() if size else None, size, stream))
    return out, lse


def attention_weights(cache: PagedKV, q, k, lse, mask=None, count=None, select=None, acc=None, scale: float | None = None):
    """The attention weight of the selected tokens on each position (tg_cuda_attn_weights).

    q, k, mask, count, scale as in tree_attention, lse as it returned it. select int64 [seqs]: the
    tokens that count, as bits (None: all). acc f32 [seqs, nkv, >= max_len]: what the cached
    positions had before (None: zeros). Returns (acc + weight [seqs, nkv, max_len], zero past a
    sequence's length; the drafted tokens' own weight [seqs, nkv, tokens])."""
    d = _drafts(cache, q, k, None, mask, count, scale)
    B, T, nq = q.shape[:3]
    dev = cache.device
    _tensor("lse", lse, torch.float32, (B, T, nq), dev)
    if select is not None:
        _tensor("select", select, torch.int64, (B,), dev)
    ab = ah = 0
    if acc is not None:
        _tensor("acc", acc, torch.float32, (B, cache.nkv, None), dev, False)
        _need(acc.shape[2] >= cache.max_len and (acc.shape[2] <= 1 or acc.stride(2) == 1), "acc: expected contiguous rows of at least max_len")
        ab, ah, _ = acc.stride()
    out = torch.empty((B, cache.nkv, cache.max_len), dtype=torch.float32, device=dev)
    fresh = torch.empty((B, cache.nkv, T), dtype=torch.float32, device=dev)
    _lib.check(_lib.lib().tg_cuda_attn_weights(cache._at, C.byref(d), lse.data_ptr(), select.data_ptr() if select is not None else None,
                                               acc.data_ptr() if acc is not None else None, ab, ah, out.data_ptr(), fresh.data_ptr(),
                                               _stream(dev)))
    return out, fresh


def commit(cache: PagedKV, k, v, count, path=None, new=None, acc=None):
    """Accepted tokens into the cache's pages (tg_cuda_kv_commit): row lens + i receives drafted row
    path[b, i] (path int32 [seqs, tokens]; None: row i) for i < count[b]. With new (the drafted tokens'
    weight from attention_weights) and acc f32 [seqs, nkv, cols], acc[b, h, lens + i] = new[b, h, path[b, i]] too.
    Returns the new lengths; the pages and acc are written in place. Any number of tokens."""
    d = _drafts(cache, None, k, v, None, count, 1.0)
    dev, T = cache.device, k.shape[1]
    if path is not None:
        _tensor("path", path, torch.int32, (cache.seqs, T), dev)
    _need((new is None) == (acc is None), "new and acc: both or neither")
    ab = ah = cols = 0
    if acc is not None:
        _tensor("new", new, torch.float32, (cache.seqs, cache.nkv, T), dev)
        _tensor("acc", acc, torch.float32, (cache.seqs, cache.nkv, None), dev, False)
        cols = acc.shape[2]
        _need(cols <= 1 or acc.stride(2) == 1, "acc: expected contiguous rows")
        ab, ah, _ = acc.stride()
    lens = torch.empty_like(cache.lens)
    _lib.check(_lib.lib().tg_cuda_kv_commit(cache._at, C.byref(d), path.data_ptr() if path is not None else None, lens.data_ptr(),
                                            new.data_ptr() if acc is not None else None, acc.data_ptr() if acc is not None else None,
                                            ab, ah, cols, _stream(dev)))
    return lens


def evict(cache: PagedKV, dst: PagedKV, acc, budget: int, recent: int = 0, sink: int = 0):
    """At most `budget` positions of each sequence and head to dst's pages, in order (tg_cuda_kv_evict):
    the first `sink`, the last `recent`, and the others with the largest acc (f32 [seqs, nkv, >= max_len]; ties:
    the lower position; NaN last). dst: pages that cache's sequences do not hold, of the same or other
    pools. Returns (kept positions int32 [seqs, nkv, budget], -1 past the last; their acc, 0 past
    the last; the lengths in dst)."""
    dev = cache.device
    _need(dst.device == dev and dst.dtype is cache.dtype, "dst: expected the cache's type and device")
    _tensor("acc", acc, torch.float32, (cache.seqs, cache.nkv, None), dev, False)
    _need(acc.shape[2] >= cache.max_len and (acc.shape[2] <= 1 or acc.stride(2) == 1), "acc: expected contiguous rows of at least max_len")
    _need(budget > 0, "budget: expected at least 1")
    shape = (cache.seqs, cache.nkv, budget)
    keep = torch.empty(shape, dtype=torch.int32, device=dev)
    out = torch.empty(shape, dtype=torch.float32, device=dev)
    lens = torch.empty_like(cache.lens)
    ab, ah, _ = acc.stride()
    _lib.check(_lib.lib().tg_cuda_kv_evict(cache._at, dst._at, acc.data_ptr(), ab, ah, budget, recent, sink, keep.data_ptr(), out.data_ptr(),
                                           lens.data_ptr(), _stream(dev)))
    return keep, out, lens
