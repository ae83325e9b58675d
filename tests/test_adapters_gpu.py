"""Low-rank adapters against the Float64 oracle.

Tolerances: a result is rounded once, half a step of its type.  Before that, sums of n products are off by n roundings of 2^-24
(tensor cores, which cut: 2^-23) of their magnitudes; scale * A * X is kept as two terms of a 16-bit type, each rounded: half a
step squared of it (Float16: and 2^-25, a half step of its smallest numbers), which the following product carries on."""
import numpy as np
import pytest
import torch

import nnlib_jl_b200 as nb
from oracle import experts_oracle as R

DEV = torch.device("cuda:0")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _cols(a, dtype=F32):
    return nb.jl_from_numpy(np.asarray(a, np.float32), device=DEV).to(dtype)


def _ints(a):
    return nb.jl_from_numpy(np.asarray(a, np.int32), device=DEV)


def _f64(t):
    return nb.jl_to_numpy(t).astype(np.float64)


def _turned(t, turn):
    """The same matrices, stored transposed."""
    if not turn:
        return t
    out = nb.jl_empty((t.shape[1], t.shape[0], *t.shape[2:]), t.dtype, t.device)
    out.copy_(t.transpose(0, 1))
    return out.transpose(0, 1)


def _close(got, want, dtype, size, what):
    got = _f64(got)
    lim = torch.finfo(dtype).eps / 2 * 1.001 * np.abs(want) + size + (2.0 ** -25 if dtype == F16 else 2.0 ** -126)
    assert got.shape == want.shape and np.isfinite(got).all(), what
    assert (np.abs(got - want) <= lim).all(), (what, float((np.abs(got - want) - lim).max()))


def _sizes(W, X, A, B, ids, offsets, scale, dtype, dY=None):
    """Bounds of what the Float32 sums and the kept A X are off by, for Y and, with dY, for dX, dA, dB."""
    u = 2.0 ** (-24 if dtype == F32 else -23)
    (M, K), r = W.shape, A.shape[0]
    half = torch.finfo(dtype).eps / 2
    kept = 0.0 if dtype == F32 else half * half * 1.01
    tiny = 2.0 ** -25 if dtype == F16 else 0.0
    W, X, A, B, scale = (np.abs(v) for v in (W, X, A, B, scale))
    mine = [(a, b, i) for (a, b), i in zip(R.runs(offsets, X.shape[1]), ids) if 0 <= i < A.shape[2]]
    y = (K + r + 4) * u * (W @ X) + ((K + r + 4) * u * 2 + kept) * R.adapters(np.zeros_like(W), X, A, B, ids, offsets, scale)
    for a, b, i in mine:
        y[:, a:b] += tiny * B[:, :, i].sum(1, keepdims=True)
    if dY is None:
        return y
    d = np.abs(dY)
    dX, dA, dB = R.adapters_back(W, X, A, B, ids, offsets, scale, d)
    dX, dA, dB = (((v + r + 4) * u * 2 + kept) * g for v, g in ((M, dX), (X.shape[1] + M, dA), (X.shape[1] + K, dB)))
    for a, b, i in mine:
        dX[:, a:b] += tiny * A[:, :, i].sum(0)[:, None]
        dA[:, :, i] += tiny * X[:, a:b].sum(1)
        dB[:, :, i] += tiny * d[:, a:b].sum(1, keepdims=True)
    return y, dX, dA, dB


CASES = [
    # M, K, r, n, lengths of the requests, the pair of each
    (128, 64, 8, 3, [10, 1, 0, 30], [0, 2, 1, -1]),
    (136, 72, 16, 4, [1] * 20, [i % 5 - 1 for i in range(20)]),
    (256, 512, 64, 2, [300, 5, 129], [1, 1, 0]),
    (300, 200, 4, 8, [17, 64, 3], [7, 0, 7]),
    (64, 1000, 128, 2, [70, 70], [1, 0]),
    (33, 35, 5, 3, [9, 40, 2], [2, 5, 0]),
    (512, 264, 32, 1, [600], [0]),
    (1, 1, 1, 1, [3], [0]),
    (264, 96, 16, 60, [1] * 64, list(range(60)) + [-1, 3, 3, 60]),
    (520, 528, 48, 5, [256, 256, 1, 255, 257, 40], [0, 1, 2, 3, 4, 0]),
    (128, 128, 100, 2, [], []),
]


@pytest.mark.gpu
@pytest.mark.parametrize("turn", [(0, 0, 0), (1, 0, 1), (0, 1, 0), (1, 1, 1)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,K,r,n,lens,ids", CASES)
def test_adapter_mul_and_its_pullback(dtype, M, K, r, n, lens, ids, turn):
    gen = np.random.default_rng(M + K + r)
    N = sum(lens)
    offsets = np.concatenate(([0], np.cumsum(lens))).astype(int)
    W, A, B = (_turned(_cols(gen.standard_normal(s) / np.sqrt(s[1]), dtype), t) for s, t in zip(((M, K), (r, K, n), (M, r, n)), turn))
    X, dY = _cols(gen.standard_normal((K, N)), dtype), _cols(gen.standard_normal((M, N)), dtype)
    scale = gen.uniform(0.5, 2.0, n)
    y, back = nb.adapter_mul_pullback(W, X, A, B, _ints(ids), offsets=_ints(offsets), scale=_cols(scale))
    dX, dA, dB = back(dY)
    assert dA.stride() == A.stride() and dB.stride() == B.stride()
    w, x, a, b, d, s = _f64(W), _f64(X), _f64(A), _f64(B), _f64(dY), np.float32(scale).astype(np.float64)
    sizes = _sizes(w, x, a, b, ids, offsets, s, dtype, d)
    _close(y, R.adapters(w, x, a, b, ids, offsets, s), dtype, sizes[0], "Y")
    for got, want, size, what in zip((dX, dA, dB), R.adapters_back(w, x, a, b, ids, offsets, s, d), sizes[1:], ("dX", "dA", "dB")):
        _close(got, want, dtype, size, what)
    assert (nb.adapter_mul(W, X, A, B, _ints(ids), offsets=_ints(offsets), scale=_cols(scale)) == y).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_requests_as_a_dimension_and_as_single_columns(dtype):
    gen = np.random.default_rng(2)
    M, K, r, n, L, B_ = 72, 40, 8, 3, 7, 5
    W, A, B = (_cols(gen.standard_normal(s) / np.sqrt(s[1]), dtype) for s in ((M, K), (r, K, n), (M, r, n)))
    X = _cols(gen.standard_normal((K, L, B_)), dtype)
    ids = [2, -1, 0, 0, 1]
    y, back = nb.adapter_mul_pullback(W, X, A, B, _ints(ids), scale=0.5)
    flat = nb.jl_reshape(X, (K, L * B_))
    y2, back2 = nb.adapter_mul_pullback(W, flat, A, B, _ints(ids), offsets=_ints(np.arange(B_ + 1) * L), scale=0.5)
    assert tuple(y.shape) == (M, L, B_) and (nb.jl_reshape(y, (M, L * B_)) == y2).all()
    dY = _cols(gen.standard_normal((M, L, B_)), dtype)
    g, g2 = back(dY), back2(nb.jl_reshape(dY, (M, L * B_)))
    assert tuple(g[0].shape) == (K, L, B_) and (nb.jl_reshape(g[0], (K, L * B_)) == g2[0]).all() and (g[1] == g2[1]).all() and (g[2] == g2[2]).all()
    each = [ids[i // L] for i in range(L * B_)]
    y3 = nb.adapter_mul(W, flat, A, B, _ints(each), scale=0.5)
    w, x, a, b = _f64(W), _f64(flat), _f64(A), _f64(B)
    s = np.full(n, 0.5)
    _close(y3, R.adapters(w, x, a, b, each, np.arange(L * B_ + 1), s), dtype, _sizes(w, x, a, b, each, np.arange(L * B_ + 1), s, dtype), "columns")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_columns_of_no_request_and_pairs_that_do_not_meet(dtype):
    """Columns before the first and behind the last request get W X; a pair, or a request, with infinities or NaN reaches no other."""
    gen = np.random.default_rng(3)
    M, K, r, n, N = 136, 64, 16, 4, 200
    W, A, B = (_cols(gen.standard_normal(s) / np.sqrt(s[1]), dtype) for s in ((M, K), (r, K, n), (M, r, n)))
    X = _cols(gen.standard_normal((K, N)), dtype)
    offsets, ids = [10, 60, 61, 150], [0, 2, 1]
    base = nb.adapter_mul(W, X, A, B, _ints(ids), offsets=_ints(offsets))
    w, x, a, b = _f64(W), _f64(X), _f64(A), _f64(B)
    s = np.ones(n)
    _close(base, R.adapters(w, x, a, b, ids, offsets, s), dtype, _sizes(w, x, a, b, ids, offsets, s, dtype), "Y")
    A[:, :, 2], B[:, :, 3] = float("nan"), float("inf")
    X[:, 70] = float("inf")
    got = nb.adapter_mul(W, X, A, B, _ints(ids), offsets=_ints(offsets))
    same = [i for i in range(N) if i not in (60, 70)]
    assert (got[:, same] == base[:, same]).all() and torch.isnan(got[:, 60]).all()


@pytest.mark.gpu
def test_two_captured_calls_replayed_in_turn():
    gen = np.random.default_rng(4)
    M, K, r, n, N = 256, 128, 16, 8, 64
    W, A, B = (_cols(gen.standard_normal(s) / np.sqrt(s[1]), BF16) for s in ((M, K), (r, K, n), (M, r, n)))
    X, ids = [_cols(gen.standard_normal((K, N)), BF16) for _ in range(2)], _ints(gen.integers(-1, n, N))
    want = [nb.adapter_mul(W, x, A, B, ids) for x in X]
    graphs, outs = [], []
    for x in X:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(nb.adapter_mul(W, x, A, B, ids))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert all((o == w).all() for o, w in zip(outs, want))
    ids.copy_(_ints(gen.integers(-1, n, N)))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert (outs[0] == nb.adapter_mul(W, X[0], A, B, ids)).all()
    nb.device_health(DEV)


@pytest.mark.gpu
def test_refusals():
    W, A, B = nb.jl_zeros((8, 16), F32, DEV), nb.jl_zeros((4, 16, 2), F32, DEV), nb.jl_zeros((8, 4, 2), F32, DEV)
    X, ids = nb.jl_zeros((16, 6), F32, DEV), _ints([0] * 6)
    nb.adapter_mul(W, X, A, B, ids)
    for bad in (lambda: nb.adapter_mul(W.half(), X, A, B, ids), lambda: nb.adapter_mul(W, X, A, B, ids.long()), lambda: nb.adapter_mul(W, X, A[0], B, ids),
                lambda: nb.adapter_mul(W, X, A, B, ids, scale=torch.ones(2, dtype=torch.float64, device=DEV)), lambda: nb.adapter_mul(W[::2, ::2], X[::2], A, B, ids)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: nb.adapter_mul(W, X, A, B, ids[:5]), lambda: nb.adapter_mul(W, X, A, B[:, :, :1], ids), lambda: nb.adapter_mul(W, X, A, B, ids, offsets=_ints([0, 6])),
                lambda: nb.adapter_mul(W, X, A, B, ids, scale=torch.ones(3, device=DEV)), lambda: nb.adapter_mul(W, nb.jl_zeros((16, 3, 2), F32, DEV), A, B, ids),
                lambda: nb.adapter_mul(W, nb.jl_zeros((16, 3, 2), F32, DEV), A, B, ids[:2], offsets=_ints([0, 3, 6])),
                lambda: nb.adapter_mul(W, X, nb.jl_zeros((130, 16, 2), F32, DEV), nb.jl_zeros((8, 130, 2), F32, DEV), ids)):
        with pytest.raises(nb.ArgumentError):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("N", [5, 700])
def test_an_infinite_column_stays_infinite(dtype, N):
    """Everything is positive, so that an infinity of X is one of its column's result, and no other's."""
    M, K, r, n = 136, 72, 8, 2
    W, A, B = (_cols(np.full(s, 0.125), dtype) for s in ((M, K), (r, K, n), (M, r, n)))
    X = _cols(np.ones((K, N)), dtype)
    X[40, 2] = float("inf")
    for how in ({}, {"offsets": _ints([0, 3, N])}):
        ids = _ints([0, 1] if how else [i % 2 for i in range(N)])
        y, back = nb.adapter_mul_pullback(W, X, A, B, ids, **how)
        assert torch.isinf(y[:, 2]).all() and torch.isfinite(y[:, :2]).all() and torch.isfinite(y[:, 3:]).all()
        dY = _cols(np.full((M, N), 0.125), dtype)
        dX, dA, dB = back(dY)
        assert torch.isinf(dB[:, :, 0]).all() and torch.isfinite(dB[:, :, 1]).all() and torch.isfinite(dX).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_empty_arrays(dtype):
    for M, K, n, N in ((0, 8, 2, 5), (8, 0, 2, 5), (8, 8, 0, 5), (8, 8, 2, 0), (0, 0, 0, 0)):
        W, A, B, X = (nb.jl_zeros(s, dtype, DEV) for s in ((M, K), (4, K, n), (M, 4, n), (K, N)))
        y, back = nb.adapter_mul_pullback(W, X, A, B, torch.zeros(N, dtype=torch.int32, device=DEV))
        assert tuple(y.shape) == (M, N) and (y == 0).all()
        for t, s in zip(back(nb.jl_zeros((M, N), dtype, DEV)), ((K, N), (4, K, n), (M, 4, n))):
            assert tuple(t.shape) == s and (t == 0).all()
    W, A, B = (nb.jl_zeros(s, dtype, DEV) for s in ((8, 8), (4, 8, 2), (8, 4, 2)))
    for L, R in ((0, 3), (3, 0)):
        y, back = nb.adapter_mul_pullback(W, torch.zeros(R, L, 8, dtype=dtype, device=DEV).permute(2, 1, 0), A, B, torch.zeros(R, dtype=torch.int32, device=DEV))
        assert tuple(y.shape) == (8, L, R) and [tuple(t.shape) for t in back(y)] == [(8, L, R), (4, 8, 2), (8, 4, 2)]
