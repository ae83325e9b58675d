"""Products of ragged groups of columns: :func:`~nnlib_jl_b200.batched_mul` for batches whose sizes a router decides on the
device.  A layer of experts is

    r = route_topk(logits, k)            # each token's k best experts, and the tokens' order by expert
    h = f.(grouped_mul(A1, x, r))        # the columns of x, gathered in that order, times their expert's matrix
    y = combine(grouped_mul(A2, h, r.offsets), r)    # back to the tokens' order, weighted

and each of the three has its pullback.  Arrays are column-major: ``x`` is ``(features, tokens)``, ``logits`` ``(experts,
tokens)``, the matrices ``(rows, features, experts)``, or ``batched_transpose`` of ``(features, rows, experts)``.  Group sizes are
read on the device only, so that a captured call follows what they are when it is replayed.  NNlib.jl has no counterpart.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Union

import torch

from . import _lib
from .attention import _DTYPES, ArgumentError, _check, _on_device, _status_word, _stream

__all__ = ["Routing", "route_topk", "route_topk_pullback", "grouped_mul", "grouped_mul_", "grouped_mul_pullback", "combine",
           "combine_pullback"]

_blank_route = bytes(_lib.RouteParams())
_blank_grouped = bytes(_lib.GroupedParams())
_blank_combine = bytes(_lib.CombineParams())


class Routing(NamedTuple):
    """What :func:`route_topk` gives for ``N`` tokens.  The chosen (token, expert) pairs are numbered by expert, then by token."""

    weights: torch.Tensor
    """``(k, N)`` Float32, in falling order of what they were chosen by"""
    experts: torch.Tensor
    """``(k, N)`` Int32, from 0; -1 for a token that takes no part"""
    offsets: torch.Tensor
    """``(G + 1)`` Int32: expert ``g`` has the numbers ``offsets[g] .. offsets[g + 1] - 1``"""
    columns: torch.Tensor
    """``(k N)`` Int32: the token of each number, -1 from ``offsets[G]`` on"""
    position: torch.Tensor
    """``(k, N)`` Int32: the number of each pair, -1 where there is none"""


def _matrix(name: str, t, like: Optional[torch.Tensor] = None) -> int:
    """Column stride of a 2-d CUDA array whose rows are adjacent."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise TypeError(f"{name} lives on {t.device}: this method is defined for CUDA arrays only")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} has eltype {t.dtype}; supported: Float16, BFloat16, Float32")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise TypeError(f"{name} must have the eltype and device of the other arrays")
    if t.ndim != 2:
        raise TypeError(f"{name} must be a 2-d (features, columns) array")
    E, N = t.shape
    if not E or not N:
        return max(E, 1)
    s0, s1 = t.stride()
    if (E > 1 and s0 != 1) or (N > 1 and s1 < E):
        raise TypeError(f"{name}: features must be adjacent and columns apart (strides {t.stride()} for size {(E, N)})")
    return s1 if N > 1 else max(E, 1)


def _factor(name: str, t: torch.Tensor):
    """(stored transposed, leading dimension, matrix stride) of a (rows, columns, matrices) array."""
    r, c, n = t.shape
    if not r or not c or not n:
        return 0, max(r, 1), 0
    s0, s1, s2 = t.stride()
    if c > 1 and s1 == 1 and (r == 1 or s0 >= c):
        trans, ld = 1, (s0 if r > 1 else c)
    elif (r <= 1 or s0 == 1) and (c <= 1 or s1 >= r):
        trans, ld = 0, (s1 if c > 1 else max(r, 1))
    elif c == 1 and s0 > 1:
        trans, ld = 1, s0                            # (a column of a matrix whose rows are adjacent)
    else:
        raise TypeError(f"{name}: rows or columns must be adjacent (strides {t.stride()} for size {tuple(t.shape)})")
    return trans, ld, (s2 if n > 1 else 0)


def _vector(name: str, t, dtype, n: Optional[int], dev) -> int:
    """Address of a dense vector on the device of the arrays."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != dev:
        raise TypeError(f"{name} must be a {str(dtype)[6:]} CUDA tensor on the device of the arrays")
    if t.ndim != 1 or (n is not None and t.shape[0] != n) or (t.shape[0] > 1 and t.stride(0) != 1):
        raise ArgumentError(f"{name} must be a dense vector{'' if n is None else f' of {n} elements'}, got size {tuple(t.shape)}")
    return t.data_ptr()


def _pairs(name: str, t, dtype, k: Optional[int], N: Optional[int], dev) -> int:
    """Address of a dense (k, N) array."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != dev:
        raise TypeError(f"{name} must be a {str(dtype)[6:]} CUDA tensor on the device of the arrays")
    if t.ndim != 2 or (k is not None and t.shape[0] != k) or (N is not None and t.shape[1] != N) \
            or (t.numel() and ((t.shape[0] > 1 and t.stride(0) != 1) or (t.shape[1] > 1 and t.stride(1) != t.shape[0]))):
        raise ArgumentError(f"{name} must be a dense column-major array of {('k' if k is None else k, 'N' if N is None else N)} elements, "
                            f"got size {tuple(t.shape)}, strides {t.stride()}")
    return t.data_ptr()


def _columns(t: torch.Tensor, E: int, N: int) -> torch.Tensor:
    """A dense column-major (E, N) array of the type and on the device of ``t``."""
    return t.new_empty_strided((E, N), (1, E or 1))


_entries: dict = {}


def _run(entry: str, p, dev, works: bool = True):
    """The library's entry point of that name, with a workspace where it wants one."""
    fns = _entries.get(entry)
    if fns is None:
        lib = _lib.load()
        fns = _entries[entry] = (getattr(lib, "nnlib_b200_" + entry), getattr(lib, f"nnlib_b200_{entry}_workspace_bytes") if works else None)
    call, size = fns
    ref = C.byref(p)
    with _on_device(dev):
        if size is None:
            _check(call(ref, _stream()), entry)
            return
        need = size(ref)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _check(call(ref, ws.data_ptr() if need else None, need, _stream()), entry)


# ------------------------------------------------------------------------------------------------- router
def _route_params(logits, k, normalize):
    p = _lib.RouteParams.from_buffer_copy(_blank_route)
    p.logits_stride = _matrix("logits", logits)
    G, N = logits.shape
    k = int(k)
    if k < 1 or k > G:
        raise ArgumentError(f"cannot choose {k} of {G} experts")
    p.dtype, p.normalize = _DTYPES[logits.dtype], 1 if normalize else 0
    p.G, p.N, p.k = G, N, k
    p.logits = logits.data_ptr()
    return p, G, N, k


def route_topk(logits: torch.Tensor, k: int, *, bias: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
               normalize: bool = True) -> Routing:
    """Each token's ``k`` largest of the ``(experts, tokens)`` logits (at most 32 of at most 1024), their softmax weights, and
    the tokens' order by expert: a :class:`Routing`.

    The weights are the softmax over the chosen (``normalize``) or, of the chosen, that over all experts.  ``bias``, Float32,
    one per expert, is added for the choice alone.  ``mask``, Bool, one per token: false takes no part.  Equal logits choose
    the lower expert first; a NaN is chosen last.  Softmax as elsewhere here: equal shares for +Inf, NaN where a NaN, or nothing but -Inf, is among
    those it is over.  Order and weights are the same each time."""
    p, G, N, k = _route_params(logits, k, normalize)
    dev = logits.device
    if bias is not None:
        p.bias = _vector("bias", bias, torch.float32, G, dev)
    if mask is not None:
        p.mask = _vector("mask", mask, torch.bool, N, dev)
    ints = torch.empty(3 * k * N + G + 1, dtype=torch.int32, device=dev)
    r = Routing(logits.new_empty_strided((k, N), (1, k), dtype=torch.float32), ints.as_strided((k, N), (1, k), 0),
                ints.as_strided((G + 1,), (1,), 3 * k * N), ints.as_strided((k * N,), (1,), k * N), ints.as_strided((k, N), (1, k), 2 * k * N))
    at = ints.data_ptr()
    p.weights, p.experts, p.columns, p.position, p.offsets = r.weights.data_ptr(), at, at + 4 * k * N, at + 8 * k * N, at + 12 * k * N
    _run("route", p, dev)
    return r


def route_topk_pullback(logits: torch.Tensor, k: int, *, bias: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                        normalize: bool = True):
    """``rrule``-style forward of :func:`route_topk`: ``(routing, back)`` where ``back(dweights)``, Float32 ``(k, N)``, gives
    the gradient of the logits.  The choice has none, and neither has ``bias``.  Logits, weights and experts are looked at
    again and may not be written to in between."""
    r = route_topk(logits, k, bias=bias, mask=mask, normalize=normalize)

    def back(dweights: torch.Tensor):
        p, G, N, k_ = _route_params(logits, k, normalize)
        p.dweights = _pairs("dweights", dweights, torch.float32, k_, N, logits.device)
        d = _columns(logits, G, N)
        p.weights, p.experts, p.dlogits = r.weights.data_ptr(), r.experts.data_ptr(), d.data_ptr()
        _run("route_bwd", p, logits.device, works=False)
        return d

    return r, back


# ------------------------------------------------------------------------------------------------- products
def _grouped(A, X, runs):
    """The struct of a product, without its result."""
    p = _lib.GroupedParams.from_buffer_copy(_blank_grouped)
    p.ldx = _matrix("X", X)
    if not isinstance(A, torch.Tensor) or A.dtype != X.dtype or A.device != X.device:
        raise TypeError("A must be a CUDA tensor of the eltype and on the device of X")
    if A.ndim != 3 or A.shape[1] != X.shape[0]:
        raise ArgumentError(f"A must be a (rows, {X.shape[0]}, matrices) array, got size {tuple(A.shape)}")
    p.transA, p.lda, p.strideA = _factor("A", A)
    M, K, G = A.shape
    N = R = X.shape[1]
    if isinstance(runs, Routing):
        p.columns = _vector("columns", runs.columns, torch.int32, None, X.device)
        R = runs.columns.shape[0]
        runs = runs.offsets
    p.offsets = _vector("offsets", runs, torch.int32, G + 1, X.device)
    p.dtype = _DTYPES[X.dtype]
    p.M, p.K, p.G, p.N, p.R = M, K, G, N, R
    p.A, p.X = A.data_ptr(), X.data_ptr()
    p.status = _status_word(X.device).data_ptr()
    return p, M, R


def grouped_mul_(Cm: torch.Tensor, A: torch.Tensor, X: torch.Tensor, runs: Union[torch.Tensor, Routing]) -> torch.Tensor:
    """:func:`grouped_mul` into ``Cm``, ``(rows, columns)`` with adjacent rows that shares no memory with
    the arguments; its columns in no run are left as they are."""
    p, M, R = _grouped(A, X, runs)
    p.ldc = _matrix("C", Cm, X)
    if tuple(Cm.shape) != (M, R):
        raise ArgumentError(f"C must be of size {(M, R)}, got {tuple(Cm.shape)}")
    p.C = Cm.data_ptr()
    _run("grouped_gemm", p, X.device)
    return Cm


def grouped_mul(A: torch.Tensor, X: torch.Tensor, runs: Union[torch.Tensor, Routing]) -> torch.Tensor:
    """``C[:, i] = A[:, :, g] * X[:, i]`` for the columns ``i`` of run ``g``: ``A`` is ``(M, K, G)``, ``X`` ``(K, N)`` with
    adjacent features, ``runs`` the ``G + 1`` Int32 offsets of the runs, ``offsets[g] .. offsets[g + 1] - 1``, on the device.
    With a :class:`Routing` the columns of ``X`` are gathered: column ``i`` of the result is of column ``routing.columns[i]``.
    Columns of the result in no run are zeros, and so are those whose column of ``X`` does not exist.  Sums are Float32, results rounded once.  Offsets beyond
    the columns count as their end; a run that ends before it begins is empty, so offsets may fall; runs must not overlap.  One matrix for all
    runs may be ``A.expand(M, K, G)``."""
    p, M, R = _grouped(A, X, runs)
    out = _columns(X, M, R)
    p.C, p.ldc, p.zero_rest = out.data_ptr(), M or 1, 1
    _run("grouped_gemm", p, X.device)
    return out


def grouped_mul_pullback(A: torch.Tensor, X: torch.Tensor, runs: Union[torch.Tensor, Routing]):
    """``rrule``-style forward of :func:`grouped_mul`: ``(C, back)`` where ``back(dC)`` gives ``(dA, dX)``.  Nothing but the
    arguments is kept, so none of them may be written to in between.  ``dA`` is stored as ``A`` is, zeros for an empty run.
    The gradients of columns that a :class:`Routing` gathers several times are rounded before they are added, in Float32, and their sum is rounded
    again: 1.4 times one rounding (Float32 ones would be twice the bytes to write and to read).  Its ``position`` must be
    that of the columns of ``X``, and the inverse of its ``columns``; pairs in no run, those of experts that are not among its offsets, add nothing."""
    out = grouped_mul(A, X, runs)
    if isinstance(runs, Routing):
        _pairs("position", runs.position, torch.int32, None, X.shape[1], X.device)

    def back(dC: torch.Tensor):
        p, M, R = _grouped(A, X, runs)
        p.ldc = _matrix("dC", dC, X)
        if tuple(dC.shape) != (M, R):
            raise ArgumentError(f"dC must be of size {(M, R)}, got {tuple(dC.shape)}")
        K, G = A.shape[1:]
        p.C = dC.data_ptr()
        dA = A.new_empty_strided((M, K, G), (K or 1, 1, M * K) if p.transA else (1, M or 1, M * K))
        p.A, p.lda, p.strideA = dA.data_ptr(), (K if p.transA else M) or 1, M * K
        _run("grouped_gemm_grad", p, X.device)
        At = A.transpose(0, 1)
        if not isinstance(runs, Routing):
            return dA, grouped_mul(At, dC, runs)
        # (zeros for the pairs of experts whose part of the offsets is not here)
        return dA, _combine(grouped_mul(At, dC, runs.offsets), runs, None, ones=True)

    return out, back


# ------------------------------------------------------------------------------------------------- combine
def _combine_params(Y, r, weights, ones=False):
    p = _lib.CombineParams.from_buffer_copy(_blank_combine)
    p.Y_stride = _matrix("Y", Y)
    dev = Y.device
    p.position = _pairs("position", r.position, torch.int32, None, None, dev)
    k, N = r.position.shape
    if not ones:
        p.weights = _pairs("weights", r.weights if weights is None else weights, torch.float32, k, N, dev)
    E, R = Y.shape
    p.dtype = _DTYPES[Y.dtype]
    p.E, p.N, p.R, p.k = E, N, R, k
    p.Y = Y.data_ptr()
    return p, E, N, R


def _combine(Y, r, weights, ones=False):
    p, E, N, R = _combine_params(Y, r, weights, ones)
    y = _columns(Y, E, N)
    if E:
        p.y = y.data_ptr()
        _run("combine", p, Y.device, works=False)
    return y


def combine(Y: torch.Tensor, r: Routing, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[:, t] = sum_j weights[j, t] * Y[:, position[j, t]]``: the columns that a routing's pairs were given, ``(E, k N)``
    with adjacent features, back in the tokens' order.  ``weights`` are the routing's own, or other Float32 ``(k, N)`` ones.
    Pairs without a position add nothing.  Sums are Float32, rounded once."""
    return _combine(Y, r, weights)


def combine_pullback(Y: torch.Tensor, r: Routing, weights: Optional[torch.Tensor] = None):
    """``rrule``-style forward of :func:`combine`: ``(y, back)`` where ``back(dy)`` gives ``(dY, dweights)``.  The routing's
    ``columns`` and ``position`` must be each other's inverse; where they are not, there is no gradient.  Nothing but the
    arguments is kept, so none of them may be written to in between."""
    y = _combine(Y, r, weights)

    def back(dy: torch.Tensor):
        p, E, N, R = _combine_params(Y, r, weights)
        p.dy_stride = _matrix("dy", dy, Y)
        if tuple(dy.shape) != (E, N):
            raise ArgumentError(f"dy must be of size {(E, N)}, got {tuple(dy.shape)}")
        p.columns = _vector("columns", r.columns, torch.int32, R, Y.device)
        dY, dw = _columns(Y, E, R), Y.new_empty_strided(r.position.shape, (1, r.position.shape[0]), dtype=torch.float32)
        if not E:
            return dY, dw.zero_()
        p.dy, p.dY, p.dweights = dy.data_ptr(), dY.data_ptr(), dw.data_ptr()
        _run("combine_bwd", p, Y.device, works=False)
        return dY, dw

    return y, back
