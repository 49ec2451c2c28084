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
import struct

import torch

from . import _lib

# tg_cuda_drafts as bytes, which ctypes passes by address: cheaper than filling a Structure each call
_pack_drafts = struct.Struct("@2if4xP3q2P3q2P").pack
assert struct.calcsize("@2if4xP3q2P3q2P") == C.sizeof(_lib.Drafts)

_TYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _int32(**values: int) -> None:
    """The library's ints: ctypes would keep the low 32 bits of more."""
    for name, x in values.items():
        _need(-(1 << 31) <= x < 1 << 31, f"{name}: {x} does not fit 32 bits")


def _check(name: str, x, dtype, shape, index: int) -> None:
    """x is a contiguous tensor of this type and shape on CUDA device `index`."""
    if x.dtype is not dtype or x.shape != shape or x.get_device() != index or not x.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous {dtype} tensor {tuple(shape)} on cuda:{index}, got {x.dtype} "
                         f"{tuple(x.shape)} strides {x.stride()} on {x.device}")


def _alike(x, y) -> bool:
    """Tensors of one shape whose strides are the same wherever there is more than one element along them."""
    return x.stride() == y.stride() or all(n == 1 or a == b for n, a, b in zip(x.shape, x.stride(), y.stride()))


def _weights(name: str, x, cache: "PagedKV", least: int) -> tuple:
    """x is f32 [seqs, nkv, >= least] on the cache's device, rows contiguous; its strides."""
    n = x.shape
    if x.dtype is not torch.float32 or x.get_device() != cache.index or len(n) != 3 or n[0] != cache.seqs or n[1] != cache.nkv or \
            n[2] < least or (n[2] > 1 and x.stride(2) != 1):
        raise ValueError(f"{name}: expected a float32 tensor [{cache.seqs}, {cache.nkv}, at least {least}] on cuda:{cache.index} with contiguous "
                         f"rows, got {x.dtype} {tuple(n)} strides {x.stride()} on {x.device}")
    return x.stride()


def _stream(cache: "PagedKV") -> int:
    """The current stream of the cache's device, which has to be the current one."""
    if cache.index != torch.cuda.current_device():
        raise ValueError(f"the cache is on cuda:{cache.index}, which is not the current device")
    return torch._C._cuda_getCurrentRawStream(cache.index)  # torch.cuda.current_stream's handle without its object


class _ForwardOnly(torch.autograd.Function):
    """out and lse as results of inputs that want a gradient: there is none, and asking for it is an error."""

    @staticmethod
    def forward(ctx, out, lse, *inputs):
        return out.detach(), lse.detach()

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("kvcache.tree_attention has no backward pass")


class PagedKV:
    """One layer's cache: pools k and v, the table of pages [seqs, cols] and lengths [seqs] (int32).

    max_len bounds every entry of lens (default: what the table holds); it sizes the launches, so a
    bound near the longest sequence is best."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, max_len: int | None = None):
        _need(k.dim() == 4 and k.dtype in _TYPES and k.is_cuda, "k: expected an f32, f16 or bf16 CUDA tensor [pages, nkv, page, head_dim]")
        _need(k.shape[3] <= 1 or k.stride(3) == 1, "k: the head dimension must be contiguous")
        _need(v.dtype is k.dtype and v.device == k.device and v.shape == k.shape and _alike(v, k),
              "v: expected k's type, device, shape and strides")
        self.index = k.get_device()
        _need(table.dim() == 2, "table: expected [seqs, cols]")
        _check("table", table, torch.int32, table.shape, self.index)
        _check("lens", lens, torch.int32, table.shape[:1], self.index)
        self.k, self.v, self.table, self.lens = k, v, table, lens
        self.device, self.dtype = k.device, k.dtype
        self.seqs, cols = table.shape
        pages, self.nkv, self.page, self.head_dim = k.shape
        self.scale = 1 / math.sqrt(self.head_dim) if self.head_dim else 1.0  # of the scores, where a call gives none
        self.max_len = self.page * cols if max_len is None else int(max_len)
        _int32(max_len=self.max_len, pages=pages, cols=cols, seqs=self.seqs)
        s = _lib.Kv(_TYPES[k.dtype], self.seqs, self.nkv, self.head_dim, self.page, pages, cols, self.max_len,
                    k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), table.data_ptr(), lens.data_ptr())
        self._struct = s
        self._at = C.addressof(s)
        self._plans = {}  # (tokens, nq) -> bytes of tree_attention's scratch, and a shape to make its lse like
        self._one = torch.empty(1, dtype=torch.float32, device=k.device)

    def with_lens(self, lens: torch.Tensor, max_len: int | None = None) -> "PagedKV":
        """The same pages with other lengths (what `commit` returned)."""
        return PagedKV(self.k, self.v, self.table, lens, max_len)


def _drafts(cache: PagedKV, q, k, v, mask, count, scale):
    """The C description of drafted tokens (tg_cuda_drafts), checked."""
    index, dt, n, dim = cache.index, cache.dtype, k.shape, cache.head_dim
    sk = k.stride()
    if k.dtype is not dt or k.get_device() != index or len(n) != 4 or n[0] != cache.seqs or n[2] != cache.nkv or n[3] != dim or sk[3] != 1:
        raise ValueError(f"k: expected a {dt} tensor [{cache.seqs}, tokens, {cache.nkv}, {dim}] on cuda:{index} with contiguous rows, got {k.dtype} "
                         f"{tuple(n)} strides {sk} on {k.device}")
    if v is not None and (v.dtype is not dt or v.get_device() != index or v.shape != n or not _alike(v, k)):
        raise ValueError(f"v: expected k's type, device, shape and strides, got {v.dtype} {tuple(v.shape)} strides {v.stride()} on {v.device}")
    nq, sq = 0, (0, 0, 0, 1)
    if q is not None:
        m, sq = q.shape, q.stride()
        if q.dtype is not dt or q.get_device() != index or len(m) != 4 or m[0] != n[0] or m[1] != n[1] or m[3] != dim or sq[3] != 1:
            raise ValueError(f"q: expected a {dt} tensor [{n[0]}, {n[1]}, heads, {dim}] on cuda:{index} with contiguous rows, got {q.dtype} "
                             f"{tuple(m)} strides {sq} on {q.device}")
        nq = m[2]
    if mask is not None:
        _check("mask", mask, torch.int64, n[:2], index)
    if count is not None:
        _check("count", count, torch.int32, n[:1], index)
    return _pack_drafts(n[1], nq, cache.scale if scale is None else scale, 0 if q is None else q.data_ptr(), sq[0], sq[1], sq[2],
                        k.data_ptr(), 0 if v is None else v.data_ptr(), sk[0], sk[1], sk[2],
                        0 if mask is None else mask.data_ptr(), 0 if count is None else count.data_ptr())


def tree_attention(cache: PagedKV, q, k, v, mask=None, count=None, scale: float | None = None):
    """Attention of drafted tokens over the cache and each other (tg_cuda_tree_attn).

    q [seqs, tokens, nq, head_dim]; k, v [seqs, tokens, nkv, head_dim], not yet in the cache; at most 64
    tokens. mask int64 [seqs, tokens]: bit u of an entry = the token attends to drafted token u (None:
    a chain). count int32 [seqs]: tokens drafted (None: all). Returns (out as q, lse f32 [seqs, tokens,
    nq]); a token that sees nothing has out 0 and lse -inf. Forward only: where q, k or v require a
    gradient, a backward pass through the results is an error (the other calls' results never require one)."""
    d = _drafts(cache, q, k, v, mask, count, scale)
    stream, shape = _stream(cache), q.shape
    plan = cache._plans.get(shape[1:3])
    if plan is None:
        size = _lib.lib().tg_cuda_tree_attn_workspace(cache._at, d)
        if size < 0:
            _lib.check(size)
        plan = cache._plans[shape[1:3]] = size, cache._one.expand(shape[:3])
    size, like = plan
    out, lse = torch.empty_like(q), torch.empty_like(like)
    # held until the kernels are launched: from then on the allocator gives its memory only to what comes after them on the stream
    work = q.new_empty(size, dtype=torch.uint8) if size else None
    so = out.stride()
    _lib.check(_lib.lib().tg_cuda_tree_attn(cache._at, d, out.data_ptr(), so[0], so[1], so[2], lse.data_ptr(),
                                            work.data_ptr() if size else None, size, stream))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _ForwardOnly.apply(out, lse, q, k, v)
    return out, lse


def attention_weights(cache: PagedKV, q, k, lse, mask=None, count=None, select=None, acc=None, scale: float | None = None):
    """The attention weight of the selected tokens on each position (tg_cuda_attn_weights).

    q, k, mask, count, scale as in tree_attention, lse as it returned it (or of any strides). select int64 [seqs]: the
    tokens that count, as bits (None: all). acc f32 [seqs, nkv, >= max_len]: what the cached
    positions had before (None: zeros). Returns (acc + weight [seqs, nkv, max_len], zero past a
    sequence's length; the drafted tokens' own weight [seqs, nkv, tokens])."""
    d = _drafts(cache, q, k, None, mask, count, scale)
    n = q.shape
    lse = lse.contiguous()  # as tree_attention gives it, or a copy
    _check("lse", lse, torch.float32, n[:3], cache.index)
    if select is not None:
        _check("select", select, torch.int64, n[:1], cache.index)
    sa = (0, 0) if acc is None else _weights("acc", acc, cache, cache.max_len)
    out = lse.new_empty((n[0], cache.nkv, cache.max_len))
    fresh = lse.new_empty((n[0], cache.nkv, n[1]))
    _lib.check(_lib.lib().tg_cuda_attn_weights(cache._at, d, lse.data_ptr(), None if select is None else select.data_ptr(),
                                               None if acc is None else acc.data_ptr(), sa[0], sa[1], out.data_ptr(), fresh.data_ptr(),
                                               _stream(cache)))
    return out, fresh


def commit(cache: PagedKV, k, v, count, path=None, new=None, acc=None):
    """Accepted tokens into the cache's pages (tg_cuda_kv_commit): row lens + i receives drafted row
    path[b, i] (path int32 [seqs, tokens]; None: row i) for i < count[b]. With new (the drafted tokens'
    weight from attention_weights) and acc f32 [seqs, nkv, cols], acc[b, h, lens + i] = new[b, h, path[b, i]] too.
    Returns the new lengths; the pages and acc are written in place. Any number of tokens."""
    d = _drafts(cache, None, k, v, None, count, 1.0)
    T = k.shape[1]
    if path is not None:
        _check("path", path, torch.int32, (cache.seqs, T), cache.index)
    _need((new is None) == (acc is None), "new and acc: both or neither")
    sa = (0, 0)
    if acc is not None:
        _check("new", new, torch.float32, (cache.seqs, cache.nkv, T), cache.index)
        sa = _weights("acc", acc, cache, 0)
    lens = torch.empty_like(cache.lens)
    _lib.check(_lib.lib().tg_cuda_kv_commit(cache._at, d, None if path is None else path.data_ptr(), lens.data_ptr(),
                                            None if acc is None else new.data_ptr(), None if acc is None else acc.data_ptr(), sa[0], sa[1],
                                            0 if acc is None else acc.shape[2], _stream(cache)))
    return lens


def evict(cache: PagedKV, dst: PagedKV, acc, budget: int, recent: int = 0, sink: int = 0):
    """At most `budget` positions of each sequence and head to dst's pages, in order (tg_cuda_kv_evict):
    the first `sink`, the last `recent`, and the others with the largest acc (f32 [seqs, nkv, >= max_len]; ties:
    the lower position; NaN last). dst: pages that cache's sequences do not hold, of the same or other
    pools. Returns (kept positions int32 [seqs, nkv, budget], -1 past the last; their acc, 0 past
    the last; the lengths in dst)."""
    _need(dst.index == cache.index and dst.dtype is cache.dtype, "dst: expected the cache's type and device")
    _need(budget > 0, "budget: expected at least 1")
    _int32(budget=budget, recent=recent, sink=sink)
    sa = _weights("acc", acc, cache, cache.max_len)
    shape = (cache.seqs, cache.nkv, budget)
    keep = cache.lens.new_empty(shape)
    out = acc.new_empty(shape)
    lens = torch.empty_like(cache.lens)
    _lib.check(_lib.lib().tg_cuda_kv_evict(cache._at, dst._at, acc.data_ptr(), sa[0], sa[1], budget, recent, sink, keep.data_ptr(), out.data_ptr(),
                                           lens.data_ptr(), _stream(cache)))
    return keep, out, lens
