"""Norm and rotation of query and key heads: what a decoder layer does to its queries and keys before
:func:`~nnlib_jl_b200.dot_product_attention`, in one pass over them, and its pullback.

Arrays are column-major like everywhere here; ``q`` is ``(nheads * d, len, batch)``, ``k`` ``(kv heads * d, len, batch)``
with features next to each other.  Both may be views into one projection's result: only the features of a token have to be
adjacent.  NNlib.jl has no counterpart.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Union

import torch

from . import _lib
from .attention import _DTYPES, ArgumentError, _check, _on_device, _stream

__all__ = ["rope_frequencies", "qk_norm_rope", "qk_norm_rope_pullback"]

_blank = bytes(_lib.NormRopeParams())


def rope_frequencies(dim: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """Angle per position of each of the ``dim / 2`` feature pairs, ``base^(-2 p / dim)``, in Float64: the ``freqs`` of
    :func:`qk_norm_rope`.  A program that stretches positions scales what this returns."""
    if dim < 0 or dim % 2:
        raise ArgumentError(f"the number of rotated features must be even, got {dim}")
    p = torch.arange(dim // 2, dtype=torch.float64)
    return (float(base) ** (-2.0 * p / max(dim, 1))).to(device)


def _require_rows(name: str, t: torch.Tensor, like: Optional[torch.Tensor] = None):
    """Strides (token, sequence) of a 3-d CUDA array whose features are adjacent; 0 where there is only one."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise TypeError(f"{name} lives on {t.device}: this method is defined for CUDA arrays only")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} has eltype {t.dtype}; supported: Float16, BFloat16, Float32")
    size = t.shape
    if len(size) != 3:
        raise TypeError(f"{name} must be a 3-d (features, length, batch) array")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise TypeError(f"{name} must have the eltype and device of the other arrays")
    E, L, B = size
    s0, sl, sb = t.stride()
    if (E > 1 and s0 != 1) or (L > 1 and sl < E) or (B > 1 and sb < 1):
        raise TypeError(f"{name}: features must be adjacent and tokens apart (strides {t.stride()} for size {tuple(size)})")
    return (sl if L > 1 else 0), (sb if B > 1 else 0)


def _dense(t: torch.Tensor, E: int, L: int, B: int) -> torch.Tensor:
    """A dense column-major (E, L, B) array of the type and on the device of ``t``."""
    s1 = E or 1
    return t.new_empty_strided((E, L, B), (1, s1, s1 * (L or 1)))


def _int32(name: str, t: torch.Tensor, n: int, dev: torch.device) -> int:
    """Address of a dense Int32 vector of n elements."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != dev:
        raise TypeError(f"{name} must be an Int32 CUDA tensor on the device of the arrays")
    if t.ndim != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        raise ArgumentError(f"{name} must be a dense vector of {n} elements, got size {tuple(t.shape)}")
    return t.data_ptr()


def _weights(name: str, g, d: int, q, dtype) -> int:
    if not isinstance(g, torch.Tensor) or g.dtype != dtype or g.device != q.device or (dtype != q.dtype and dtype != torch.float32):
        raise TypeError(f"the {name} weights must be a CUDA vector of the arrays' eltype, or Float32, both alike")
    if g.ndim != 1 or g.shape[0] != d or (d > 1 and g.stride(0) != 1):
        raise ArgumentError(f"the {name} weights must be a dense vector of {d} elements")
    return g.data_ptr()


def _params(q, k, gq, gk, freqs, nheads, start, positions, eps, interleaved):
    qs = _require_rows("query", q)
    ks = _require_rows("key", k, q)
    Eq, L, B = q.shape
    Ek, Lk, Bk = k.shape
    nheads = int(nheads)
    if nheads < 1 or Eq % nheads != 0 or Eq == 0:
        raise ArgumentError(f"First dimension of query must be divisible by `nheads`: size {tuple(q.shape)}, nheads {nheads}")
    d = Eq // nheads
    if Lk != L or Bk != B or Ek % d != 0 or Ek == 0:
        raise ArgumentError(f"query of size {tuple(q.shape)} and key of size {tuple(k.shape)} do not match for heads of {d} features")
    p = _lib.NormRopeParams.from_buffer_copy(_blank)
    wdtype = getattr(gq, "dtype", None)
    p.gq, p.gk = _weights("query", gq, d, q, wdtype), _weights("key", gk, d, q, wdtype)
    dev = q.device
    if not isinstance(freqs, torch.Tensor) or freqs.dtype != torch.float64 or freqs.device != dev:
        raise TypeError("freqs must be a Float64 CUDA vector (rope_frequencies makes one)")
    n = freqs.shape[0] if freqs.ndim == 1 else -1
    if n < 0 or 2 * n > d or (n > 1 and freqs.stride(0) != 1):
        raise ArgumentError(f"freqs must be a dense vector of at most {d // 2} elements, got {tuple(freqs.shape)}")
    p.dtype, p.wdtype = _DTYPES[q.dtype], _DTYPES[wdtype]
    if interleaved:
        p.interleaved = 1
    p.d, p.rot, p.Hq, p.Hk, p.L, p.B = d, 2 * n, nheads, Ek // d, L, B
    p.q, p.k, p.freqs = q.data_ptr(), k.data_ptr(), freqs.data_ptr()
    p.q_stride_l, p.q_stride_b = qs
    p.k_stride_l, p.k_stride_b = ks
    p.eps = eps
    if positions is not None:
        if not isinstance(positions, torch.Tensor) or positions.dtype != torch.int32 or positions.device != dev:
            raise TypeError("positions must be an Int32 CUDA tensor on the device of the arrays")
        if tuple(positions.shape) not in ((L, B), (L,)):
            raise ArgumentError(f"positions must be of size {(L, B)} or {(L,)}, got {tuple(positions.shape)}")
        p.positions = positions.data_ptr()
        p.positions_stride = (C.c_int64 * 2)(positions.stride(0), positions.stride(1) if positions.ndim == 2 else 0)
    elif isinstance(start, torch.Tensor):
        p.start = _int32("start", start, B, dev)
    else:
        p.start0 = int(start)
    return p


def qk_norm_rope(q, k, gq, gk, freqs, *, nheads: int, start: Union[int, torch.Tensor] = 0,
                 positions: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False):
    """RMS norm of every head of ``q`` and ``k`` and the rotation of its features by position: returns ``(q', k')``.

    Each head's ``d = size(q, 1) / nheads`` features ``x`` become ``n = x / sqrt(mean(x^2) + eps) * g`` with the weights
    ``gq`` / ``gk`` (``d`` elements, of the arrays' element type or Float32); then pair ``p`` of its first
    ``2 * length(freqs)`` features is turned by the angle ``position * freqs[p]`` — features ``p`` and
    ``p + length(freqs)``, or ``2p`` and ``2p + 1`` where ``interleaved``; the others stay as they are.  Token ``l`` of
    sequence ``b`` is at position ``start + l``, ``start`` an integer or an Int32 tensor of one per sequence, or at
    ``positions[l, b]`` (Int32; ``(len,)`` serves every sequence; ``start`` is not looked at then).  ``k`` has as many heads as
    its size says.  Arithmetic is Float32 (angles in 64 bits until they are less than a turn; sines and cosines to
    2^-21 where all results are 16-bit), results are rounded once; head sizes are even, up to 256."""
    p = _params(q, k, gq, gk, freqs, nheads, start, positions, eps, interleaved)
    yq, yk = _dense(q, *q.shape), _dense(k, *k.shape)
    p.yq, p.yk = yq.data_ptr(), yk.data_ptr()
    with _on_device(q.device):
        _check(_lib.load().nnlib_b200_norm_rope(C.byref(p), _stream()), "norm_rope")
    return yq, yk


def qk_norm_rope_pullback(q, k, gq, gk, freqs, *, nheads: int, start: Union[int, torch.Tensor] = 0,
                          positions: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False):
    """``rrule``-style forward of :func:`qk_norm_rope`: returns ``(q', k', back)`` where ``back(dq', dk')`` gives
    ``(dq, dk, dgq, dgk)``.  Nothing but the arguments is kept, so none of them (``start`` and ``positions`` among them) may
    be written to in between.
    The gradients of the weights are summed in Float32 in a fixed order and rounded to the weights' element type."""
    yq, yk = qk_norm_rope(q, k, gq, gk, freqs, nheads=nheads, start=start, positions=positions, eps=eps, interleaved=interleaved)

    def back(dyq: torch.Tensor, dyk: torch.Tensor):
        p = _params(q, k, gq, gk, freqs, nheads, start, positions, eps, interleaved)
        for name, t, like in (("dq", dyq, q), ("dk", dyk, k)):
            strides = _require_rows(name, t, like)
            if t.shape != like.shape:
                raise ArgumentError(f"{name} must have size {tuple(like.shape)}, got {tuple(t.shape)}")
            if name == "dq":
                p.dyq, (p.dyq_stride_l, p.dyq_stride_b) = t.data_ptr(), strides
            else:
                p.dyk, (p.dyk_stride_l, p.dyk_stride_b) = t.data_ptr(), strides
        dq, dk = _dense(q, *q.shape), _dense(k, *k.shape)
        dgq, dgk = torch.empty_like(gq), torch.empty_like(gk)
        p.dq, p.dk, p.dgq, p.dgk = dq.data_ptr(), dk.data_ptr(), dgq.data_ptr(), dgk.data_ptr()
        lib = _lib.load()
        with _on_device(q.device):
            need = lib.nnlib_b200_norm_rope_bwd_workspace_bytes(C.byref(p))
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
            _check(lib.nnlib_b200_norm_rope_bwd(C.byref(p), ws.data_ptr(), need, _stream()), "norm_rope_bwd")
        return dq, dk, dgq, dgk

    return yq, yk, back
