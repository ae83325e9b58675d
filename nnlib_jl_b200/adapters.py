"""Low-rank adapters of many requests beside a shared matrix: a server multiplies the tokens of all requests by one ``W``, each
request's own correction of it being a pair of thin matrices; a program that trains such pairs leaves ``W`` as it is.

Arrays are column-major.  ``X`` is ``(K, N)``, all requests' columns one after the other, or ``(K, L, requests)``; ``W`` is ``(M, K)``, the pairs are
``A`` ``(r, K, n)`` and ``B`` ``(M, r, n)``, each stored as it is or as its transpose (``transpose(0, 1)`` of it).  NNlib.jl has
no counterpart.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Union

import torch

from . import _lib
from .attention import _DTYPES, ArgumentError, _status_word
from .experts import _columns, _factor, _matrix, _run, _vector
from .layout import is_column_major

__all__ = ["adapter_mul", "adapter_mul_pullback"]

_blank = bytes(_lib.AdapterParams())


def _flat(name: str, X, like=None):
    """A (features, columns) view of X and the columns of a request, or None where X has but columns."""
    if isinstance(X, torch.Tensor) and X.ndim == 3:
        if X.numel() and not is_column_major(X):
            raise TypeError(f"{name}: a 3-d array must be dense and column-major (strides {X.stride()} for size {tuple(X.shape)})")
        L = X.shape[1]
        X = X.as_strided((X.shape[0], L * X.shape[2]), (1, X.shape[0] or 1))
        _matrix(name, X, like)
        return X, L
    _matrix(name, X, like)
    return X, None


def _params(W, X, A, B, adapters, offsets, scale):
    p = _lib.AdapterParams.from_buffer_copy(_blank)
    X2, L = _flat("X", X)
    p.ldx = _matrix("X", X2)
    dev, (K, N) = X2.device, X2.shape
    for name, t, dims in (("W", W, 2), ("A", A, 3), ("B", B, 3)):
        if not isinstance(t, torch.Tensor) or t.dtype != X2.dtype or t.device != dev:
            raise TypeError(f"{name} must be a CUDA tensor of the eltype and on the device of X")
        if t.ndim != dims:
            raise TypeError(f"{name} must have {dims} dimensions, got {t.ndim}")
    M, (r, n) = W.shape[0], (A.shape[0], A.shape[2])
    if W.shape[1] != K or A.shape[1] != K or tuple(B.shape) != (M, r, n):
        raise ArgumentError(f"W of size {tuple(W.shape)}, A of size {tuple(A.shape)}, B of size {tuple(B.shape)} and X of size "
                            f"{tuple(X.shape)} do not match")
    if r < 1 or r > 128:
        raise ArgumentError(f"rank {r}: from 1 to 128 are supported")
    p.dtype = _DTYPES[X2.dtype]
    p.transW, p.ldw, _ = _factor("W", W.unsqueeze(2))
    p.transA, p.lda, p.strideA = _factor("A", A)
    p.transB, p.ldb, p.strideB = _factor("B", B)
    p.M, p.K, p.N, p.r, p.n = M, K, N, r, n
    p.W, p.A, p.B, p.X = W.data_ptr(), A.data_ptr(), B.data_ptr(), X2.data_ptr()
    if offsets is not None:
        if L is not None:
            raise ArgumentError("offsets are for a 2-d X; the requests of a 3-d one are its last dimension")
        p.ids = _vector("adapters", adapters, torch.int32, None, dev)
        p.runs = adapters.shape[0]
        p.offsets = _vector("offsets", offsets, torch.int32, p.runs + 1, dev)
    else:
        p.run_len = 1 if L is None else L
        p.runs = N if L is None else X.shape[2]
        p.ids = _vector("adapters", adapters, torch.int32, p.runs, dev)
    if isinstance(scale, torch.Tensor):
        p.scale = _vector("scale", scale, torch.float32, n, dev)
    else:
        p.scale0 = scale
    p.status = _status_word(dev).data_ptr()
    return p, X2


def _shaped(out: torch.Tensor, X: torch.Tensor) -> torch.Tensor:
    return out if X.ndim == 2 else out.as_strided((out.shape[0], *X.shape[1:]), (1, out.shape[0] or 1, (out.shape[0] or 1) * (X.shape[1] or 1)))


def adapter_mul(W: torch.Tensor, X: torch.Tensor, A: torch.Tensor, B: torch.Tensor, adapters: torch.Tensor, *,
                offsets: Optional[torch.Tensor] = None, scale: Union[float, torch.Tensor] = 1.0) -> torch.Tensor:
    """``W * X + scale[a] * B[:, :, a] * (A[:, :, a] * X)``, ``a`` being the pair of the request that a column belongs to:
    ``adapters``, Int32, one per request, from 0; one outside the pairs (-1, say) has none and gets ``W * X``.

    The requests are the last dimension of a 3-d ``X``.  For a 2-d one they are runs of columns, ``offsets[b] .. offsets[b + 1]
    - 1`` (Int32, one more than requests, on the device; a column in no run gets ``W * X``; a run that ends before it begins is empty; runs must not
    overlap), or, without ``offsets``, single columns.  More than 1024 requests with ``offsets`` are computed on the CUDA cores, at a thirtieth of the
    rate: without them, or as a 3-d ``X``, they are not.  ``scale``: a number, or Float32, one per pair.  Ranks from 1 to 128.  Pairs may share a
    matrix (``expand``).

    Both terms are summed in Float32 and rounded once.  In between, ``scale * A * X`` is kept as two terms of the element type or in Float32 (few
    columns).  With Float16 arrays it may so be infinite beyond 65504, whatever ``B`` makes of it, and is off by up to 2^-25, half a step of the smallest
    numbers, which makes 2^-25 of the magnitudes in a row of ``B``.  Infinities and NaN of a pair are in the columns of its requests alone."""
    p, X2 = _params(W, X, A, B, adapters, offsets, scale)
    out = _columns(X2, W.shape[0], X2.shape[1])
    p.C, p.ldc = out.data_ptr(), W.shape[0] or 1
    _run("adapter_gemm", p, X2.device)
    return _shaped(out, X)


def adapter_mul_pullback(W: torch.Tensor, X: torch.Tensor, A: torch.Tensor, B: torch.Tensor, adapters: torch.Tensor, *,
                         offsets: Optional[torch.Tensor] = None, scale: Union[float, torch.Tensor] = 1.0):
    """``rrule``-style forward of :func:`adapter_mul`: ``(Y, back)`` where ``back(dY)`` gives ``(dX, dA, dB)``; ``W`` is taken
    as fixed.  ``dA`` and ``dB`` are stored as ``A`` and ``B`` are, zeros for a pair that no request names; requests that
    share a pair add to it in their order.  They take ``scale * A * X`` and ``scale * B' * dY`` with 16 (BFloat16) or 22 bits, in Float16 down to
    2^-36.  Nothing but the arguments is kept, so none of them may be written to in between."""
    y = adapter_mul(W, X, A, B, adapters, offsets=offsets, scale=scale)

    def back(dY: torch.Tensor):
        p, X2 = _params(W, X, A, B, adapters, offsets, scale)
        if tuple(dY.shape) != tuple(y.shape):
            raise ArgumentError(f"dY must be of size {tuple(y.shape)}, got {tuple(dY.shape)}")
        d2, _ = _flat("dY", dY, X2)
        (M, K), (r, n) = W.shape, (A.shape[0], A.shape[2])
        dX = _columns(X2, K, X2.shape[1])
        dA = A.new_empty_strided((r, K, n), (K or 1, 1, r * K) if p.transA else (1, r, r * K))
        dB = B.new_empty_strided((M, r, n), (r, 1, M * r) if p.transB else (1, M or 1, M * r))
        p.dC, p.lddc = d2.data_ptr(), _matrix("dY", d2)
        p.dX, p.dA, p.dB = dX.data_ptr(), dA.data_ptr(), dB.data_ptr()
        _run("adapter_bwd", p, X2.device)
        return _shaped(dX, X), dA, dB

    return y, back
