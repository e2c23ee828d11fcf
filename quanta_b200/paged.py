"""Paged KV cache: append with rotation, attention over pages, attention behind a shared prefix.

The serving counterparts of ``decoder.rope_append`` and ``decoder.sdpa_decode`` for batches whose sequences have
different lengths: keys and values live in pages of one pool, sequences name their pages in a table, several query
heads may share a K/V head, and a call takes single tokens, drafts, prompts or chunks of prompts, mixed.  (The
reference's attention is one dense block of equal lengths, ``crates/ml/quanta-nn/src/kernel.rs:64-175``.)

Lengths and page numbers stay on the device: a call that was captured in a CUDA graph follows what the tensors hold
when it is replayed.  What cannot be checked on the host (a length past the table, a page number outside the pool) is
recorded on the device and raised by ``PagedKVCache.check``.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import numpy as np
import torch

from . import _lib as L
from .quant import QuantError, check as _check

# The pieces of torch.cuda.device / current_stream that cost 0.1 us instead of 1.5 and 2 (a decode step makes dozens of calls).
_device_now = getattr(torch._C, "_cuda_getDevice", None)
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None)

_DTYPE = {torch.float32: L.F32, torch.bfloat16: L.BF16, torch.float16: L.F16}


def _bad(message: str, code: int = L.ERR_INVALID_PARAM):
    raise QuantError(code, message)


def _want(ok: bool, message: str, code: int = L.ERR_INVALID_PARAM):
    if not ok:
        raise QuantError(code, message)


def rope_table(n_pos: int, rot_dim: int, base: float = 10000.0, device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin of positions 0 .. n_pos - 1, ``[n_pos, rot_dim / 2]`` float32; the angles are computed in float64
    (``crates/sci/quanta-array/src/autograd/rope.rs:43-63``)."""
    theta = np.arange(n_pos, dtype=np.float64)[:, None] * np.power(float(base), -2.0 * np.arange(rot_dim // 2, dtype=np.float64) / float(rot_dim))
    return tuple(torch.from_numpy(f(theta).astype(np.float32)).to(device) for f in (np.cos, np.sin))


class PagedKVCache:
    """Two pools of pages, ``k`` and ``v``, ``[n_pages, kv_heads, page_size, head_dim]`` in bf16 or f16."""

    def __init__(self, n_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.bfloat16, device="cuda"):
        shape = (n_pages, kv_heads, page_size, head_dim)
        self._bind(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))

    @staticmethod
    def from_parts(k: torch.Tensor, v: torch.Tensor) -> "PagedKVCache":
        """A cache over existing pools (kept, not copied)."""
        c = PagedKVCache.__new__(PagedKVCache)
        c._bind(k, v)
        return c

    def _bind(self, k, v):
        _want(k.dim() == 4 and k.shape == v.shape, "PagedKVCache: two pools [n_pages, kv_heads, page_size, head_dim]", L.ERR_RANK)
        _want(k.dtype == v.dtype and k.dtype in (torch.bfloat16, torch.float16), "PagedKVCache: bf16 or f16 pools", L.ERR_NOT_SUPPORTED)
        _want(k.is_contiguous() and v.is_contiguous(), "PagedKVCache: the pools must be contiguous")
        _want(k.device == v.device, "PagedKVCache: the pools must be on one device")
        n_pages, kv_heads, page_size, head_dim = k.shape
        _want(n_pages > 0 and kv_heads > 0, "PagedKVCache: empty pools")
        _want(page_size in (16, 32, 64, 128, 256), f"PagedKVCache: page size 16, 32, 64, 128 or 256, got {page_size}", L.ERR_NOT_SUPPORTED)
        _want(head_dim in (64, 128), f"PagedKVCache: head dim 64 or 128, got {head_dim}", L.ERR_NOT_SUPPORTED)
        self.k, self.v, self.device, self.dtype = k, v, k.device, k.dtype
        self.n_pages, self.kv_heads, self.page_size, self.head_dim = n_pages, kv_heads, page_size, head_dim
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        self.c = L.PagedKv(k.data_ptr(), v.data_ptr(), self.status.data_ptr(), n_pages, page_size, kv_heads, head_dim, _DTYPE[k.dtype])
        self._ref = ctypes.byref(self.c)
        self._index = k.device.index if k.is_cuda else -1
        self._scale = 1.0 / math.sqrt(head_dim)
        self._f32 = torch.empty(0, dtype=torch.float32, device=k.device)  # new_empty of a tensor is the quickest allocation

    def check(self) -> None:
        """Waits for the current stream and raises what a kernel recorded (once)."""
        _run(self, L.load().qb200_paged_check, self._ref)


class PagedBatch:
    """Which pages and how many keys each sequence of a call has: ``table [batch, width]``, ``kv_lens [batch]`` (the
    call's new tokens included) and, unless every sequence has exactly one new token, ``cu_q [batch + 1]`` (sequence b's
    new tokens are rows ``cu_q[b]:cu_q[b + 1]`` of the call's arrays; rows outside ``cu_q[0]:cu_q[batch]`` belong to nobody and are
    left as they are in every output); int32 on the cache's device.  The tensors are kept, so their contents may change
    between calls (in stream order: not while a call that reads them runs); a batch can be used for the whole life of a set of slots."""

    def __init__(self, cache: PagedKVCache, table: torch.Tensor, kv_lens: torch.Tensor, cu_q: Optional[torch.Tensor] = None):
        _want(table.dim() == 2 and kv_lens.dim() == 1 and (cu_q is None or cu_q.dim() == 1), "PagedBatch: table [batch, width], kv_lens [batch], cu_q [batch + 1]",
              L.ERR_RANK)
        b, width = table.shape
        _want(b > 0 and width > 0, "PagedBatch: an empty table", L.ERR_LENGTH)
        _want(kv_lens.shape[0] == b and (cu_q is None or cu_q.shape[0] == b + 1), "PagedBatch: kv_lens or cu_q does not match the table's rows", L.ERR_LENGTH)
        for t in (table, kv_lens) if cu_q is None else (table, kv_lens, cu_q):
            _want(t.dtype == torch.int32 and t.device == cache.device and t.stride(-1) == 1, "PagedBatch: int32 tensors on the cache's device, rows contiguous")
        _want(b == 1 or table.stride(0) >= width, "PagedBatch: the table's rows overlap")
        self.cache, self.table, self.kv_lens, self.cu_q, self.size = cache, table, kv_lens, cu_q, b
        self.c = L.PagedBatch(table.data_ptr(), kv_lens.data_ptr(), 0 if cu_q is None else cu_q.data_ptr(), max(table.stride(0), width), width, b)
        self._ref = ctypes.byref(self.c)
        self._floats = {}  # scratch sizes by shape of the call


def _run(cache: PagedKVCache, fn, *args) -> None:
    """fn(*args, stream) with the cache's device current, on its current stream."""
    index = cache._index
    if index < 0:
        _bad("the cache is not on a CUDA device", L.ERR_CUDA)
    if _device_now is not None and _stream_of is not None and _device_now() == index:
        status = fn(*args, _stream_of(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, torch.cuda.current_stream(index).cuda_stream)
    if status:
        _check(status)


def _rows(x: torch.Tensor, heads: int, cache: PagedKVCache, what: str) -> Tuple[int, int, int]:
    """(tokens, heads, row stride) of x ``[tokens, heads * head_dim]`` with contiguous columns; heads = 0: as many as there are."""
    shape = x.shape
    if len(shape) == 2:
        tokens, width = shape
        step, col = x.stride()
        n = width // cache.head_dim
        if n and n * cache.head_dim == width and (n == heads or heads == 0) and col == 1 and x.get_device() == cache._index:
            return tokens, n, step if tokens > 1 else width  # (one row has no next one)
    if x.device != cache.device:
        _bad(f"{what} is on {x.device}, the cache on {cache.device}")
    _bad(f"{what} must be [tokens, {heads or 'heads'} * {cache.head_dim}] with contiguous columns, got {list(shape)}", L.ERR_LENGTH)


def _small(x: torch.Tensor, dtype, n: int, device, what: str) -> int:
    if x.dtype != dtype or x.dim() != 1 or x.shape[0] != n or x.device != device or not x.is_contiguous():
        _bad(f"{what} must be {n} contiguous {dtype} values on {device}")
    return x.data_ptr()


def paged_rope_append(batch: PagedBatch, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                      positions: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes the new tokens' keys (rotated) and values into their sequences' pages and returns the rotated queries in
    the cache's type.  ``q [tokens, heads * head_dim]``, ``k``, ``v [tokens, kv_heads * head_dim]`` in f32, bf16 or f16
    (all the same; rows may be strided, such as the parts of a fused projection); ``cos``, ``sin [n_pos, rot_dim / 2]``
    from ``rope_table``; ``positions [tokens]`` int32 (default: the token's place in its sequence).  q may be None."""
    cache = batch.cache
    dev = cache.device
    tokens, _, ks = _rows(k, cache.kv_heads, cache, "paged_rope_append: k")
    v_tokens, _, vs = _rows(v, cache.kv_heads, cache, "paged_rope_append: v")
    q_tokens, heads, qs = (tokens, 0, 0) if q is None else _rows(q, 0, cache, "paged_rope_append: q")
    if not v_tokens == tokens == q_tokens:
        _bad("paged_rope_append: q, k and v differ in tokens", L.ERR_LENGTH)
    x_dtype = _DTYPE.get(k.dtype)
    if x_dtype is None or v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
        _bad("paged_rope_append: q, k and v must be f32, bf16 or f16, all the same", L.ERR_NOT_SUPPORTED)
    table = cos.shape
    if not (len(table) == 2 and table == sin.shape and cos.dtype is sin.dtype is torch.float32 and cos.is_contiguous() and sin.is_contiguous() and
            cos.get_device() == sin.get_device() == cache._index):
        _bad("paged_rope_append: cos and sin must be contiguous f32 [n_pos, rot_dim / 2] on the cache's device")
    pos = 0 if positions is None else _small(positions, torch.int32, tokens, dev, "paged_rope_append: positions")
    if q is None:
        _want(q_out is None, "paged_rope_append: q_out without q")
    elif q_out is None:
        q_out = cache.k.new_empty(tokens, heads * cache.head_dim)
    else:
        _want(q_out.shape == q.shape and q_out.dtype == cache.dtype and q_out.device == dev and q_out.is_contiguous(),
              "paged_rope_append: q_out must be contiguous, of q's shape and the cache's type")
    _run(cache, L.load().qb200_paged_rope_append, cache._ref, batch._ref, 0 if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(), x_dtype, qs, ks, vs,
         tokens, heads, cos.data_ptr(), sin.data_ptr(), 2 * table[1], table[0], pos, 0 if q is None else q_out.data_ptr())
    return q_out


def _attend(who: str, batch: PagedBatch, q: torch.Tensor, slopes, out, lse):
    """The checks that both attentions share: (tokens, heads, q's row stride, pointer of slopes, out, pointer of lse)."""
    cache = batch.cache
    dev = cache.device
    tokens, heads, qs = _rows(q, 0, cache, who)
    if q.dtype != cache.dtype:
        _bad(f"{who}: q is {q.dtype}, the cache {cache.dtype}", L.ERR_NOT_SUPPORTED)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != cache.dtype or out.device != dev or not out.is_contiguous():
        _bad(f"{who}: out must be contiguous, of q's shape and the cache's type")
    if lse is not None and (lse.shape != (tokens, heads) or lse.dtype != torch.float32 or lse.device != dev or not lse.is_contiguous()):
        _bad(f"{who}: lse must be contiguous f32 [{tokens}, {heads}]")
    return tokens, heads, qs, 0 if slopes is None else _small(slopes, torch.float32, heads, dev, who + ": slopes"), out, 0 if lse is None else lse.data_ptr()


def _scratch(who: str, batch: PagedBatch, scratch: Optional[torch.Tensor], size_of, *shape) -> Optional[torch.Tensor]:
    """The call's workspace: the caller's, or one of its own from torch's allocator (which keeps calls on different
    streams and in different captured graphs apart), or None where it needs none."""
    cache = batch.cache
    floats = batch._floats.get(shape)
    if floats is None:
        if cache._index < 0:
            _bad("the cache is not on a CUDA device", L.ERR_CUDA)
        if len(batch._floats) >= 1024:
            batch._floats.clear()
        with torch.cuda.device(cache._index):
            floats = batch._floats[shape] = size_of(cache._ref, batch._ref, *shape)
    if scratch is None:
        return cache._f32.new_empty(floats) if floats else None
    if scratch.dtype != torch.float32 or scratch.device != cache.device or not scratch.is_contiguous() or scratch.numel() < floats:
        _bad(f"{who}: scratch must be {floats} contiguous f32 values on {cache.device}", L.ERR_LENGTH)
    return scratch


def paged_attention(batch: PagedBatch, q: torch.Tensor, scale: Optional[float] = None, softcap: float = 0.0, slopes: Optional[torch.Tensor] = None,
                    prefix_lens: Optional[torch.Tensor] = None, causal: bool = True, out: Optional[torch.Tensor] = None,
                    lse: Optional[torch.Tensor] = None, scratch: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Every new token against its sequence's keys: ``q [tokens, heads * head_dim]`` of the cache's type -> the same shape.
    A token sees the keys up to its own place (``causal``), and the first ``prefix_lens[b]`` keys of its sequence where
    that is given (int32 ``[batch]``).  ``scale`` defaults to 1 / sqrt(head_dim); ``softcap`` > 0 caps the scores by
    ``softcap * tanh(score / softcap)``; ``slopes [heads]`` f32 subtract ``slopes[h] * distance``.  ``lse [tokens, heads]``
    f32 receives the log of each row's sum of exp(score).  A row that sees no key gives zeros and -inf."""
    cache = batch.cache
    tokens, heads, qs, sl, out, lp = _attend("paged_attention", batch, q, slopes, out, lse)
    pl = 0 if prefix_lens is None else _small(prefix_lens, torch.int32, batch.size, cache.device, "paged_attention: prefix_lens")
    lib = L.load()
    scratch = _scratch("paged_attention", batch, scratch, lib.qb200_paged_attention_scratch_floats, tokens, heads)
    _run(cache, lib.qb200_paged_attention, cache._ref, batch._ref, q.data_ptr(), qs, tokens, heads, cache._scale if scale is None else scale, softcap, sl, pl,
         1 if causal else 0, 0 if scratch is None else scratch.data_ptr(), out.data_ptr(), lp)
    return out


def shared_prefix_attention(batch: PagedBatch, q: torch.Tensor, prefix_pages: torch.Tensor, prefix_len: int, scale: Optional[float] = None,
                            softcap: float = 0.0, slopes: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                            lse: Optional[torch.Tensor] = None, scratch: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``paged_attention`` for a batch whose sequences all begin with the same ``prefix_len`` keys, kept once in the pages
    ``prefix_pages`` (int32): the batch's table and lengths name what follows the prefix, and the prefix is read once for
    all tokens.  A token's place counts from the prefix's first key."""
    cache = batch.cache
    tokens, heads, qs, sl, out, lp = _attend("shared_prefix_attention", batch, q, slopes, out, lse)
    if prefix_len <= 0:
        _bad("shared_prefix_attention: the prefix is empty (call paged_attention)")
    need = -(-prefix_len // cache.page_size)
    if prefix_pages.dim() != 1 or prefix_pages.dtype != torch.int32 or not prefix_pages.is_contiguous() or prefix_pages.get_device() != cache._index or \
            prefix_pages.shape[0] < need:
        _bad(f"shared_prefix_attention: {prefix_len} keys need {need} contiguous int32 page numbers on {cache.device}", L.ERR_LENGTH)
    lib = L.load()
    scratch = _scratch("shared_prefix_attention", batch, scratch, lib.qb200_shared_prefix_scratch_floats, prefix_len, tokens, heads)
    _run(cache, lib.qb200_shared_prefix_attention, cache._ref, batch._ref, prefix_pages.data_ptr(), prefix_len, q.data_ptr(), qs, tokens, heads,
         cache._scale if scale is None else scale, softcap, sl, 0 if scratch is None else scratch.data_ptr(), out.data_ptr(), lp)
    return out
