"""A key / value cache held in 8 bits, and attention over it: the serving side of
:func:`~nnlib_jl_b200.dot_product_attention`, whose keys and values a program otherwise keeps in 16 bits.

A :class:`QuantizedCache` is a pool of pages of ``page`` tokens; one scale for every page and head, of keys and of values,
says what a code stands for.  :func:`cache_write_` quantises new tokens into it, :func:`cache_read` reads tokens back,
:func:`cached_attention` attends to it without doing so.  Sequences find their pages through a table
(``table[l // page, b]`` is the page of token ``l`` of sequence ``b``); without one, sequence ``b`` of ``batch`` owns the
``b``-th run of ``pages / batch`` pages, and calls are for ``batch`` sequences.

All of it is asynchronous on the current stream, allocates through torch and reads lengths, starts and tables on the device,
so that a captured call follows what they hold when it is replayed.  NNlib.jl has no counterpart.
"""
from __future__ import annotations

import ctypes as C
import operator
from typing import Optional, Union

import torch

from . import _lib
from .attention import _DTYPES, ArgumentError, _check, _empty3, _on_device, _status_word, _stream
from .layout import is_column_major, jl_empty
from .rotary import _dense, _int32, _require_rows

__all__ = ["QuantizedCache", "cache_write_", "cache_read", "cached_attention"]

_CODES = {torch.int8: _lib.INT8, torch.float8_e4m3fn: _lib.E4M3}
_blank_cache = bytes(_lib.Cache())
_blank_tokens = bytes(_lib.CacheTokens())
_blank_attn = bytes(_lib.CacheAttnParams())


def _fixed(slot: str) -> property:
    """An attribute of a cache: calls go by the addresses that the first arrays had, so it cannot be replaced."""
    get = operator.attrgetter(slot)

    def put(self, value):
        if value is not get(self):                     # (`cache.k_scale *= 2` assigns the same array)
            raise AttributeError(f"{slot[1:]} of a cache cannot be replaced; from_arrays makes another cache")
    return property(get, put)


class QuantizedCache:
    """Keys and values of ``nheads`` heads of ``dim / nheads`` features in 8 bits: ``capacity`` tokens (rounded up to whole
    pages) for each of ``batch`` sequences, or, for programs that hand pages out themselves, ``batch=1`` and as many tokens
    as the pool is to hold.  A call without a table is for exactly ``batch`` sequences, or refused; with a table it is for as
    many as that has.

    ``eltype``: ``torch.int8`` (a block's largest magnitude becomes 127) or ``torch.float8_e4m3fn`` (its scale is a power of
    two, the smallest that brings the largest magnitude to 448 or less).  ``page``: tokens of a page, a power of two from 16
    to 256.  The head size is a multiple of 16, at most 256.

    Arrays, all column-major: ``k`` and ``v`` codes ``(dim, page, pages)``, ``k_scale`` and ``v_scale`` Float32
    ``(nheads, pages)``; an element stands for ``code * scale``.  They can be written to, not replaced.  :meth:`from_arrays`
    takes them from elsewhere."""

    __slots__ = ("_k", "_v", "_k_scale", "_v_scale", "_batch", "_template")

    k, v, k_scale, v_scale, batch = (_fixed(name) for name in ("_k", "_v", "_k_scale", "_v_scale", "_batch"))

    def __init__(self, dim: int, capacity: int, batch: int = 1, *, nheads: int, page: int = 64, eltype=torch.int8,
                 device="cuda"):
        dim, capacity, batch, nheads, page = int(dim), int(capacity), int(batch), int(nheads), int(page)
        if page < 16 or page > 256 or page & (page - 1):
            raise ArgumentError(f"a page holds a power of two from 16 to 256 tokens, got {page}")
        if nheads < 1 or dim < 1 or dim % nheads != 0 or capacity < 0 or batch < 0:
            raise ArgumentError(f"no cache of {dim} features in {nheads} heads, {capacity} tokens and {batch} sequences")
        if eltype not in _CODES:
            raise TypeError(f"codes of type {eltype}; supported: Int8, Float8 E4M3")
        pages = batch * -(-capacity // page)
        k = jl_empty((dim, page, pages), eltype, device)
        v = jl_empty((dim, page, pages), eltype, device)
        k_scale, v_scale = jl_empty((nheads, pages), torch.float32, device), jl_empty((nheads, pages), torch.float32, device)
        for t in (k.view(torch.uint8), v.view(torch.uint8), k_scale, v_scale):
            t.zero_()
        self._set(k, v, k_scale, v_scale, batch)

    @classmethod
    def from_arrays(cls, k, v, k_scale, v_scale, *, batch: Optional[int] = None) -> "QuantizedCache":
        """The cache that these arrays make up (no copy).  Without ``batch`` it is a pool: a call without a table deals its
        pages out in equal runs to however many sequences the call is for."""
        c = cls.__new__(cls)
        c._set(k, v, k_scale, v_scale, None if batch is None else int(batch))
        return c

    def _set(self, k, v, k_scale, v_scale, batch):
        if k.dtype not in _CODES or v.dtype != k.dtype:
            raise TypeError(f"codes of types {k.dtype} and {v.dtype}; supported: Int8, Float8 E4M3, both alike")
        if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise TypeError("scales must be Float32")
        dev = k.device
        if not k.is_cuda or v.device != dev or k_scale.device != dev or v_scale.device != dev:
            raise TypeError("a cache's arrays must be on one CUDA device")
        if k.ndim != 3 or k.shape != v.shape or k_scale.ndim != 2 or k_scale.shape != v_scale.shape \
                or k_scale.shape[1] != k.shape[2] or k_scale.shape[0] < 1 or k.shape[0] % k_scale.shape[0] != 0:
            raise ArgumentError(f"codes of sizes {tuple(k.shape)} and {tuple(v.shape)} and scales of sizes {tuple(k_scale.shape)} "
                                f"and {tuple(v_scale.shape)} do not make up a cache")
        E, T, P = k.shape
        H = k_scale.shape[0]
        codes, scales = (1, E, E * T), (1, H)
        for t, strides in ((k, codes), (v, codes), (k_scale, scales), (v_scale, scales)):
            if t.stride() != strides and not is_column_major(t):       # (the first says it at a glance)
                raise TypeError("a cache's arrays must be dense and column-major")
        if T < 16 or T > 256 or T & (T - 1):
            raise ArgumentError(f"a page holds a power of two from 16 to 256 tokens, got {T}")
        if batch is not None and batch < 0:
            raise ArgumentError(f"batch = {batch}")
        self._k, self._v, self._k_scale, self._v_scale, self._batch = k, v, k_scale, v_scale, batch
        p = _lib.Cache.from_buffer_copy(_blank_cache)
        p.code = _CODES[k.dtype]
        p.d, p.H, p.page, p.pages = E // H, H, T, P
        p.k_codes, p.v_codes = k.data_ptr(), v.data_ptr()
        p.k_scale, p.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
        self._template = p

    @property
    def device(self):
        return self._k.device

    @property
    def nheads(self) -> int:
        return self._k_scale.shape[0]

    @property
    def page(self) -> int:
        return self._k.shape[1]

    @property
    def pages(self) -> int:
        return self._k.shape[2]

    def __repr__(self):
        return f"QuantizedCache(dim={self._k.shape[0]}, nheads={self.nheads}, {self.pages} pages of {self.page} tokens, {self._k.dtype})"

    def _call(self, B: int, table: Optional[torch.Tensor]):
        """The struct of a call for B sequences."""
        p = _lib.Cache.from_buffer_copy(self._template)
        p.B = B
        if table is None:
            # (a call for no sequence touches nothing)
            if B != self._batch and self._batch is not None and B:
                raise ArgumentError(f"a call for {B} sequences, without a table, on a cache of {self._batch}")
            p.rows = self._k.shape[2] // B if B else 0
            return p
        if not isinstance(table, torch.Tensor) or table.dtype != torch.int32 or table.device != self._k.device:
            raise TypeError("table must be an Int32 CUDA tensor on the cache's device")
        rows = table.shape[0]
        if table.ndim != 2 or table.shape[1] != B or (rows > 1 and table.stride(0) != 1) or (B > 1 and table.stride(1) < max(rows, 1)):
            raise ArgumentError(f"table must be a column-major array of (pages, {B}), got size {tuple(table.shape)}, strides {table.stride()}")
        p.table, p.rows = table.data_ptr(), rows
        p.table_stride = table.stride(1) if B > 1 else 0
        return p


def _starts(p, start, B, dev):
    if isinstance(start, torch.Tensor):
        p.start = _int32("start", start, B, dev)
    else:
        p.start0 = int(start)


def cache_write_(cache: QuantizedCache, k: torch.Tensor, v: torch.Tensor, *, start: Union[int, torch.Tensor] = 0,
                 count: Optional[torch.Tensor] = None, table: Optional[torch.Tensor] = None) -> QuantizedCache:
    """Quantises the tokens of ``k`` and ``v``, ``(dim, len, batch)`` arrays with adjacent features, into ``cache``: token
    ``l`` of sequence ``b`` becomes its token number ``start[b] + l`` (``start``: an integer, or Int32, one per sequence).
    With ``count`` (Int32, one per sequence) only the first ``count[b]`` tokens are written.

    A page begun by this call gets the scale that its tokens ask for; one that holds tokens before ``start`` keeps its own
    unless the new tokens need a larger one, in which case the older codes are rounded to that.  What a page holds behind the
    new tokens is left as it is; tokens beyond the capacity or on pages that the pool does not have are left out, like a
    sequence whose start is negative.  A block that is given a NaN or an infinity reads as NaN until its page is begun anew.  Pages that are
    written must be one sequence's alone."""
    kst = _require_rows("key", k)
    vst = _require_rows("value", v, k)
    if k.device != cache._k.device:
        raise TypeError(f"key lives on {k.device}, the cache on {cache._k.device}")
    E, L, B = k.shape
    if E != cache._k.shape[0] or v.shape != k.shape:
        raise ArgumentError(f"key and value must both be ({cache._k.shape[0]}, len, batch) arrays. Instead:\n"
                            f"- size(k): {tuple(k.shape)}\n- size(v): {tuple(v.shape)}")
    c = cache._call(B, table)
    p = _lib.CacheTokens.from_buffer_copy(_blank_tokens)
    p.dtype, p.L = _DTYPES[k.dtype], L
    p.k, p.v = k.data_ptr(), v.data_ptr()
    p.k_stride_l, p.k_stride_b = kst
    p.v_stride_l, p.v_stride_b = vst
    _starts(p, start, B, k.device)
    if count is not None:
        p.count = _int32("count", count, B, k.device)
    with _on_device(k.device):
        _check(_lib.load().nnlib_b200_cache_write(C.byref(c), C.byref(p), _stream()), "cache_write")
    return cache


def cache_read(cache: QuantizedCache, length: int, *, start: Union[int, torch.Tensor] = 0,
               lens: Optional[torch.Tensor] = None, table: Optional[torch.Tensor] = None, dtype=torch.bfloat16):
    """``(k, v)``: tokens ``start[b] .. start[b] + length - 1`` of every sequence as dense ``(dim, length, batch)`` arrays of
    ``dtype``, ``code * scale`` rounded once.  Tokens from ``lens[b]`` on (Int32; without it, from the capacity on) come as
    zeros, tokens on pages that the pool does not have as NaN.  The batch is the table's, else that of ``start`` or ``lens``,
    else the cache's own, or one of a pool that has none."""
    length = int(length)
    if length < 0:
        raise ArgumentError(f"length = {length}")
    if dtype not in _DTYPES:
        raise TypeError(f"eltype {dtype}; supported: Float16, BFloat16, Float32")
    B = 1 if cache._batch is None else cache._batch
    if table is not None:
        if not isinstance(table, torch.Tensor) or table.ndim != 2:
            raise TypeError("table must be a 2-d Int32 CUDA tensor")
        B = table.shape[1]
    elif isinstance(start, torch.Tensor):
        B = start.numel()
    elif isinstance(lens, torch.Tensor):
        B = lens.numel()
    dev, E = cache._k.device, cache._k.shape[0]
    c = cache._call(B, table)
    p = _lib.CacheTokens.from_buffer_copy(_blank_tokens)
    _starts(p, start, B, dev)
    if lens is not None:
        p.lens = _int32("lens", lens, B, dev)
    size, strides = (E, length, B), (1, E, E * (length or 1))
    k, v = (cache._k_scale.new_empty_strided(size, strides, dtype=dtype) for _ in range(2))
    p.dtype, p.L, p.k, p.v = _DTYPES[dtype], length, k.data_ptr(), v.data_ptr()
    with _on_device(dev):
        _check(_lib.load().nnlib_b200_cache_read(C.byref(c), C.byref(p), _stream()), "cache_read")
    return k, v


def cached_attention(q: torch.Tensor, cache: QuantizedCache, lens: Union[int, torch.Tensor], *, nheads: int,
                     table: Optional[torch.Tensor] = None, start: Optional[torch.Tensor] = None, causal: bool = True,
                     scale: Optional[float] = None, return_lse: bool = False):
    """Attention of ``q``, ``(nheads * d, len, batch)`` with adjacent features, over the first ``lens[b]`` tokens of each
    sequence in ``cache`` (an integer, or Int32, one per sequence; at most the capacity counts): ``x`` of the size of ``q``, and
    with ``return_lse`` the Float32 ``(len, nheads, batch)`` log-sum-exp of each query's logits.

    Causal: query ``i`` of sequence ``b`` is at position ``start[b] + i`` (Int32; by default ``lens[b] - len + i``, the
    queries of the last tokens) and sees the tokens up to its own.  ``nheads`` is a multiple of the cache's heads; a group of
    ``nheads / cache.nheads`` query heads shares one.  ``scale`` multiplies the logits, ``1/sqrt(d)`` by default.  A query
    that sees nothing gives NaN, like one with a token among those it sees whose page the pool does not have, or whose block
    was given a NaN.

    What the call knows of lengths in a tensor is the capacity, the table's rows or the cache's: kernels are chosen and the
    workspace is sized by it.  A program that holds little in a table for much gets the kernels for much; an integer ``lens``, or a
    table of the rows in use, tells."""
    qst = _require_rows("query", q)
    dev = q.device
    if dev != cache._k.device:
        raise TypeError(f"query lives on {dev}, the cache on {cache._k.device}")
    E, L, B = q.shape
    nheads, t = int(nheads), cache._template
    if nheads < 1 or nheads % t.H != 0 or E != nheads * t.d:
        raise ArgumentError(f"query of size {tuple(q.shape)} in {nheads} heads does not match a cache of {t.H} heads of {t.d} features")
    c = cache._call(B, table)
    p = _lib.CacheAttnParams.from_buffer_copy(_blank_attn)
    p.dtype, p.causal = _DTYPES[q.dtype], 1 if causal else 0
    p.Hq, p.L = nheads, L
    if isinstance(lens, torch.Tensor):
        p.lens = _int32("lens", lens, B, dev)
    else:
        p.len0 = int(lens)
    if start is not None:
        p.start = _int32("start", start, B, dev)
    if scale is not None:
        p.scale = scale
        if not p.scale > 0:            # (as Float32, where 0 would stand for the default)
            raise ArgumentError(f"scale = {scale}")
    x = _dense(q, E, L, B)
    p.q, p.x = q.data_ptr(), x.data_ptr()
    p.q_stride_l, p.q_stride_b = qst
    lse = None
    if return_lse:
        lse = _empty3(L, nheads, B, torch.float32, dev)
        p.lse = lse.data_ptr()
    p.status = _status_word(dev).data_ptr()
    lib = _lib.load()
    with _on_device(dev):
        need = lib.nnlib_b200_cache_attn_workspace_bytes(C.byref(c), C.byref(p))
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _check(lib.nnlib_b200_cache_attn(C.byref(c), C.byref(p), ws.data_ptr() if need else None, need, _stream()), "cache_attn")
    return (x, lse) if return_lse else x
