"""A decoder's key/value cache in pages, over libtgcuda: rotary positions, new tokens into the cache with the
norm and rotation on the way, attention of drafted tokens (also below prefixes that sequences share), the attention
weight each position receives, the commit of accepted tokens, and eviction by that weight.

The pools are torch CUDA tensors [pages, nkv, page, head_dim] (any strides, rows contiguous) in f32,
f16 or bf16; position p of sequence b is row p % page of page table[b, p // page]. Everything is
asynchronous on the current stream; results are new tensors, except that `append` and `commit` write the cache's
pages (and `acc`) and `evict` the destination's. No reference counterpart: the reference recomputes
every position's keys and values (examples/qwen3/import.py:90-132).

A speculative decode step: draft tokens and their mask, `tree_attention` in every layer, compare
with the model's own choices, `commit` the accepted path. When the cache is full, `evict` by the
weights that `attention_weights` has summed up (examples/speculative.py runs all of it). A plain one: `append`
the token's projection with keys=True, then `tree_attention` or `shared_attention` over the lengths from before
with the rotated q and k; `append` alone takes a prompt into the cache."""
from __future__ import annotations

import ctypes as C
import math
import struct

import torch
from torch.autograd import forward_ad

from . import _lib

# tg_cuda_drafts as bytes, which ctypes passes by address: cheaper than filling a Structure each call
_pack_drafts = struct.Struct("@2if4xP3q2P3q2P").pack
assert struct.calcsize("@2if4xP3q2P3q2P") == C.sizeof(_lib.Drafts)

_pack_rotary = struct.Struct("@3if2Pq").pack
assert struct.calcsize("@3if2Pq") == C.sizeof(_lib.Rotary)

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
    if cache.index != torch._C._cuda_getDevice():
        raise ValueError(f"the cache is on cuda:{cache.index}, which is not the current device")
    return torch._C._cuda_getCurrentRawStream(cache.index)  # torch.cuda.current_stream's handle without its object


def _stream_of(index: int) -> int:
    """The same for tensors of a call that has no cache."""
    if index != torch._C._cuda_getDevice():
        raise ValueError(f"the tensors are on cuda:{index}, which is not the current device")
    return torch._C._cuda_getCurrentRawStream(index)


def _tangent(*tensors) -> bool:
    """Whether one of the tensors carries a tangent of forward-mode differentiation."""
    return forward_ad._current_level >= 0 and any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in tensors)


def _no_tangent(name: str, *tensors) -> None:
    """Called within a level of forward mode only."""
    if _tangent(*tensors):
        raise RuntimeError(f"kvcache.{name} has no forward-mode derivative")


def _versions(*tensors) -> tuple:
    """Those of the tensors that autograd counts the writes of: not those made in inference mode."""
    return tuple(x for x in tensors if not x.is_inference())


def _written(*tensors) -> None:
    """Autograd learns that the library has written these in place: what was saved of them for a backward pass is not used then."""
    torch.autograd.graph.increment_version(_versions(*tensors))


def _pages_written(cache) -> None:
    """The same for a cache's pools, in one call."""
    pools = getattr(cache, "_versioned", ())
    if pools:
        torch._C._increment_version(pools)


class _ForwardOnly(torch.autograd.Function):
    """out and lse as results of inputs that want a gradient: there is none, and asking for it is an error."""

    @staticmethod
    def forward(ctx, out, lse, *inputs):
        return out.detach(), lse.detach()

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("kvcache.tree_attention has no backward pass")


class _NoGradient(torch.autograd.Function):
    """The first n of the tensors as results of the others, as above, for the call of this name."""

    @staticmethod
    def forward(ctx, name, n, *tensors):
        ctx.name = name
        return tuple(x.detach() for x in tensors[:n])

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"kvcache.{ctx.name} has no backward pass")


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
        self._versioned = _versions(k, v)
        self._one = torch.empty(1, dtype=torch.float32, device=k.device)

    def with_lens(self, lens: torch.Tensor, max_len: int | None = None) -> "PagedKV":
        """The same pages with other lengths (what `commit` or `append` returned)."""
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
    gradient, a backward pass through the results is an error, and so is a tangent of theirs (attention_weights', commit's and evict's
    results never require a gradient and have no tangents)."""
    if forward_ad._current_level >= 0:
        _no_tangent("tree_attention", q, k, v)
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


class SharedPrefix:
    """Which sequences of a cache begin with the same pages (tg_cuda_prefix): made once, when the batch's composition changes.

    groups: (first sequence, sequences, shared positions) of each, ascending; sequences in none share nothing. The tables of a group's sequences
    name the same pages for the shared positions. max_own: about how many positions a sequence has at most behind what it
    shares (default: what max_len leaves); it only sizes the launches, and the lengths may grow past it. always: share even where
    tree_attention's way, a prefix read for each sequence, is faster (few sequences, short prefixes). Like any input, it has to live as long as a
    CUDA graph that was captured with it."""

    def __init__(self, cache: PagedKV, groups, max_own: int | None = None, always: bool = False):
        groups = [tuple(int(x) for x in g) for g in groups]
        end, which = 0, [-1] * cache.seqs
        for i, (first, members, shared) in enumerate(groups):
            _need(first >= end and members > 0 and first + members <= cache.seqs, f"groups: sequences {first} to {first + members - 1} of {cache.seqs}, after {end - 1}")
            _need(0 <= shared <= cache.page * cache.table.shape[1], f"groups: {shared} shared positions, of {cache.page * cache.table.shape[1]} that a table holds")
            end = first + members
            which[first:end] = [i] * members
        self.groups, self.seqs, self.index = groups, cache.seqs, cache.index
        lengths = [g[2] for g in groups]
        self.max_shared = max(lengths, default=0)
        if max_own is None:
            max_own = cache.max_len - (min(lengths) if groups and -1 not in which else 0)
        _need(max_own >= 0, f"max_own: {max_own}")
        _int32(max_own=max_own)
        made = torch.tensor([g[0] for g in groups] + [g[1] for g in groups] + lengths + which, dtype=torch.int32).to(cache.device)
        n, at = len(groups), made.data_ptr()
        self._held, self._stream = made, torch._C._cuda_getCurrentRawStream(cache.index) if made.is_cuda else 0
        self._struct = _lib.Prefix(n, self.max_shared, max_own, bool(always), at, at + 4 * n, at + 8 * n, at + 12 * n)
        self._at = C.addressof(self._struct)
        self._sizes = n, self.max_shared, max_own, bool(always)  # all that the scratch's size depends on


def shared_attention(cache: PagedKV, prefix: SharedPrefix, q, k, v, mask=None, count=None, scale: float | None = None):
    """tree_attention for a batch whose sequences share prefixes, each read once for its whole group (tg_cuda_shared_attn).

    Arguments and results as for tree_attention. Its scratch has two f32 rows for each row of q."""
    if prefix.index != cache.index or prefix.seqs != cache.seqs or prefix.max_shared > cache.max_len:
        raise ValueError(f"prefix: made for {prefix.seqs} sequences with up to {prefix.max_shared} positions shared on cuda:{prefix.index}, not for {cache.seqs} of "
                         f"up to {cache.max_len} on cuda:{cache.index}")
    if forward_ad._current_level >= 0:
        _no_tangent("shared_attention", q, k, v)
    d = _drafts(cache, q, k, v, mask, count, scale)
    stream, shape = _stream(cache), q.shape
    key = shape[1], shape[2], prefix._sizes
    plan = cache._plans.get(key)
    if plan is None:
        size = _lib.lib().tg_cuda_shared_attn_workspace(cache._at, d, prefix._at)
        if size < 0:
            _lib.check(size)
        if len(cache._plans) >= 64:  # a long-lived cache sees many batches
            cache._plans.clear()
        plan = cache._plans[key] = size, cache._one.expand(shape[:3])
    size, like = plan
    out, lse = torch.empty_like(q), torch.empty_like(like)
    work = q.new_empty(size, dtype=torch.uint8) if size else None  # held until the kernels are launched, as above
    if stream != prefix._stream:  # the prefix may be dropped while this stream's kernels have yet to read it
        prefix._held.record_stream(torch.cuda.current_stream(cache.index))
    so = out.stride()
    _lib.check(_lib.lib().tg_cuda_shared_attn(cache._at, d, prefix._at, out.data_ptr(), so[0], so[1], so[2], lse.data_ptr(),
                                              work.data_ptr() if size else None, size, stream))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _NoGradient.apply("shared_attention", 2, out, lse, q, k, v)
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
    _pages_written(cache)
    if acc is not None:
        _written(acc)
    return lens


def rotary_frequencies(part: int, theta: float = 1e4, factor: float = 1.0, original: int | None = None, fast: float = 32.0,
                       slow: float = 1.0) -> torch.Tensor:
    """Radians per position of each pair of a rotation of `part` elements, f64 on the CPU: theta^(-2 i / part).

    factor: how much longer the context is than the one a model was trained on. Without `original` every frequency is
    divided by it. With `original`, that context's length, pairs that turn `fast` times or more in it keep theirs, pairs that turn
    `slow` times or less are divided, and in between the two are mixed in proportion to the logarithm of the turns."""
    _need(part >= 0 and part % 2 == 0, f"part: expected an even number of elements, got {part}")
    _need(theta > 0 and factor > 0, "theta and factor: expected positive numbers")
    f = float(theta) ** (-2 * torch.arange(part // 2, dtype=torch.float64) / max(part, 1))
    if original is None or factor == 1:
        return f / factor
    _need(original > 0 and fast > slow > 0, "original, fast, slow: expected positive numbers, fast above slow")
    keep = (torch.log(original * f / (2 * math.pi * slow)) / math.log(fast / slow)).clamp(0, 1)
    return f * (keep + (1 - keep) / factor)


class Rotary:
    """A rotation of heads of head_dim elements by position (tg_cuda_rotary): its frequencies, on the device, and its form.

    freq: f64 [part / 2] radians per position, a CUDA tensor; None: rotary_frequencies(part, theta) on the current device. part: leading
    elements of a head that turn (default: two for each frequency, or the whole head). interleaved: neighbours 2 i and
    2 i + 1 are partners, else i and i + part / 2. gain: a factor of the turned elements."""

    def __init__(self, head_dim: int, freq: torch.Tensor | None = None, theta: float = 1e4, part: int | None = None, gain: float = 1.0,
                 interleaved: bool = False):
        if freq is None:
            freq = rotary_frequencies(head_dim if part is None else part, theta).cuda()
        _need(not freq.requires_grad, "freq: no gradient reaches the frequencies; give them detached")
        _need(freq.dim() == 1 and freq.dtype is torch.float64 and freq.is_cuda and freq.is_contiguous(), "freq: expected a contiguous float64 CUDA tensor [part / 2]")
        self.part = 2 * freq.shape[0]
        _need(part is None or part == self.part, f"part: {part} elements, but {freq.shape[0]} frequencies")
        _need(0 < head_dim <= 256 and self.part <= head_dim, f"{self.part} elements of a head of {head_dim} turn")
        self.freq, self.head_dim, self.gain, self.interleaved, self.index = freq, head_dim, float(gain), bool(interleaved), freq.get_device()
        self._at = freq.data_ptr()

    def _pack(self, pos, seqs: int, tokens: int, index: int, dim: int, inverse: bool = False) -> bytes:
        """The C description for these positions, int32 [seqs, tokens] or [tokens] (None: the call's own), checked."""
        if index != self.index or dim != self.head_dim:
            raise ValueError(f"rotary: made for heads of {self.head_dim} on cuda:{self.index}, not of {dim} on cuda:{index}")
        at, row = 0, 0
        if pos is not None:
            n = pos.shape
            if pos.dtype is not torch.int32 or pos.get_device() != index or n not in ((seqs, tokens), (tokens,)) or (tokens > 1 and pos.stride(-1) != 1):
                raise ValueError(f"pos: expected an int32 tensor [{seqs}, {tokens}] or [{tokens}] on cuda:{index} with contiguous rows, got {pos.dtype} "
                                 f"{tuple(n)} strides {pos.stride()} on {pos.device}")
            at, row = pos.data_ptr(), pos.stride(0) if len(n) == 2 else 0
        return _pack_rotary(self.part, self.interleaved, inverse, self.gain, self._at, at, row)


def _turn(x, rotary, pos, inverse, out):
    n, s, index = x.shape, x.stride(), x.get_device()
    if x.dtype not in _TYPES or len(n) != 4 or (n[3] > 1 and s[3] != 1) or index < 0:
        raise ValueError(f"x: expected an f32, f16 or bf16 CUDA tensor [seqs, tokens, heads, head_dim] with contiguous rows, got {x.dtype} {tuple(n)} "
                         f"strides {s} on {x.device}")
    r = rotary._pack(pos, n[0], n[1], index, n[3], inverse)
    if out is None:
        out = torch.empty_like(x)
    elif out.dtype is not x.dtype or out.get_device() != index or out.shape != n or (n[3] > 1 and out.stride(3) != 1):
        raise ValueError(f"out: expected x's type, shape and device and contiguous rows, got {out.dtype} {tuple(out.shape)} strides {out.stride()} on {out.device}")
    elif out.data_ptr() == x.data_ptr() and not _alike(out, x):
        raise ValueError("out: x's memory with other strides")
    o = out.stride()
    _lib.check(_lib.lib().tg_cuda_rope(r, _TYPES[x.dtype], n[0], n[1], n[2], n[3], x.data_ptr(), s[0], s[1], s[2], out.data_ptr(), o[0], o[1], o[2],
                                       _stream_of(index)))
    return out


def _rows(x):
    """x, or a copy of it whose rows are contiguous and begin on 16-byte boundaries, as the library wants them."""
    e = x.element_size()
    if (x.shape[3] > 1 and x.stride(3) != 1) or x.data_ptr() % 16 or any(n > 1 and s * e % 16 for n, s in zip(x.shape[:3], x.stride())):
        return x.clone(memory_format=torch.contiguous_format)  # (contiguous() gives x itself where only its beginning is off)
    return x


class _Rope(torch.autograd.Function):
    """A rotation's gradient is the rotation by the negative angle, with the same gain, and its derivative along a tangent is the tangent's
    rotation. any_layout: of a gradient or tangent, whose rows may lie anyhow."""

    @staticmethod
    def forward(ctx, x, rotary, pos, inverse, any_layout):
        ctx.rotary, ctx.inverse, ctx.given = rotary, inverse, pos is not None
        # the frequencies too, so that their change before the backward pass is an error (those made in inference mode have no version)
        saved = (() if pos is None else (pos,)) + (() if rotary.freq.is_inference() else (rotary.freq,))
        ctx.save_for_backward(*saved)
        ctx.save_for_forward(*saved)
        return _turn(_rows(x) if any_layout else x, rotary, pos, inverse, None)

    @staticmethod
    def backward(ctx, grad):
        return _along(ctx, grad, not ctx.inverse), None, None, None, None

    @staticmethod
    def jvp(ctx, tangent, *others):
        return _along(ctx, tangent, ctx.inverse)


def _along(ctx, x, inverse):
    """A gradient or tangent rotated to _Rope's positions."""
    saved = ctx.saved_tensors
    pos = saved[0] if ctx.given else None
    if (torch.is_grad_enabled() and x.requires_grad) or _tangent(x):
        return _Rope.apply(x, ctx.rotary, pos, inverse, True)
    return _turn(_rows(x), ctx.rotary, pos, inverse, None)


def rope(x, rotary: Rotary, pos=None, inverse: bool = False, out=None):
    """x [seqs, tokens, heads, head_dim] rotated to its tokens' positions (tg_cuda_rope); pos int32 [seqs, tokens] or [tokens] (None: 0, 1, ...).

    inverse: by the negative angle. out: where to (x itself: in place; else memory that x does not share). Differentiable with respect to
    x in reverse and forward mode, without out."""
    if (torch.is_grad_enabled() and x.requires_grad) or _tangent(x, out):
        _need(out is None, "out: not with a gradient or a tangent")
        return _Rope.apply(x, rotary, pos, inverse, False)
    if out is not None and torch.is_grad_enabled() and out.requires_grad:
        raise ValueError("out: requires a gradient, but the call's writes are not part of its history")
    y = _turn(x, rotary, pos, inverse, out)
    if out is not None:
        _written(out)
    return y


def append(cache: PagedKV, k, v, q=None, rotary: Rotary | None = None, pos=None, count=None, q_norm=None, k_norm=None, eps: float = 1e-6,
           keys: bool = False):
    """New tokens into the cache's pages, normed and rotated on the way (tg_cuda_kv_append).

    k, v [seqs, tokens, nkv, head_dim] and q [seqs, tokens, nq, head_dim]: a projection's output, any number of tokens; count int32
    [seqs]: tokens there are (None: all). Cache row lens + i receives token i's k, rotated to its position (pos, None: lens + i), and v. q_norm, k_norm
    f32 [head_dim]: weights of an RMS norm of each head before the rotation. keys: return the rotated keys too, with k's strides (and so the memory
    that k's projection spans), which tree_attention and shared_attention take with v as the tokens' own, the lengths being those from before. Returns (the new lengths, q rotated or
    None, k rotated or None), rows past count 0; the pages are written in place. Forward only, like tree_attention."""
    if forward_ad._current_level >= 0:
        _no_tangent("append", q, k, v, q_norm, k_norm)
    d = _drafts(cache, q, k, v, None, count, 1.0)
    n, dim, index = k.shape, cache.head_dim, cache.index
    qn = kn = qo = ko = qp = kp = r = None
    sq = sk = (0, 0, 0)
    if q_norm is not None:
        _check("q_norm", q_norm, torch.float32, (dim,), index)
        _need(q is not None, "q_norm: without q")
        qn = q_norm.data_ptr()
    if k_norm is not None:
        _check("k_norm", k_norm, torch.float32, (dim,), index)
        kn = k_norm.data_ptr()
    if rotary is not None:
        r = rotary._pack(pos, n[0], n[1], index, dim)
    elif pos is not None:
        raise ValueError("pos: without a rotation")
    lens = torch.empty_like(cache.lens)
    if q is not None:
        qo = torch.empty_like(q)
        sq, qp = qo.stride(), qo.data_ptr()
    if keys:
        sk = k.stride()  # v's, so that the two are drafted rows together
        ko = k.new_empty_strided(n, sk) if 0 not in sk else torch.empty_like(k)
        sk, kp = ko.stride(), ko.data_ptr()
    _lib.check(_lib.lib().tg_cuda_kv_append(cache._at, d, r, qn, kn, eps, qp, sq[0], sq[1], sq[2], kp, sk[0], sk[1], sk[2], lens.data_ptr(), _stream(cache)))
    _pages_written(cache)
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or (q is not None and q.requires_grad) or
                                    (q_norm is not None and q_norm.requires_grad) or (k_norm is not None and k_norm.requires_grad)):
        made = [x for x in (qo, ko) if x is not None]
        if made:
            made = list(_NoGradient.apply("append", len(made), *made, *(x for x in (q, k, v, q_norm, k_norm) if x is not None)))
            qo, ko = made.pop(0) if qo is not None else None, made.pop(0) if ko is not None else None
    return lens, qo, ko


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
    _pages_written(dst)
    return keep, out, lens
