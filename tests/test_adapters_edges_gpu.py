"""Calls of low-rank adapters that their documentation allows and that went wrong once: a factor that all pairs share, pairs with infinities or
NaN beside other requests', small Float16 numbers, offsets that fall, many requests.  Tolerances as in test_adapters_gpu.py."""
import numpy as np
import pytest
import torch

import nnlib_jl_b200 as nb
from oracle import experts_oracle as R
from test_adapters_gpu import BF16, DEV, F16, F32, _close, _cols, _f64, _ints, _sizes, _turned


def _factors(gen, M, K, r, n, dtype, turn=(0, 0, 0)):
    return (_turned(_cols(gen.standard_normal(s) / np.sqrt(s[1]), dtype), t) for s, t in zip(((M, K), (r, K, n), (M, r, n)), turn))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("turn", [(0, 0, 0), (0, 1, 1)])
@pytest.mark.parametrize("M,K,r,N", [(136, 72, 16, 700), (137, 67, 8, 700), (512, 264, 40, 1100), (264, 128, 16, 60)])
def test_a_factor_that_all_pairs_share(dtype, turn, M, K, r, N):
    """One matrix of stride 0 for every pair, its gradient pair by pair."""
    gen = np.random.default_rng(M + N)
    n = 5
    W, A, B = _factors(gen, M, K, r, n, dtype, turn)
    A1, B1 = (_turned(_cols(gen.standard_normal(s) / np.sqrt(s[1]), dtype), t) for s, t in zip(((r, K, 1), (M, r, 1)), turn[1:]))
    X, dY = _cols(gen.standard_normal((K, N)), dtype), _cols(gen.standard_normal((M, N)), dtype)
    ids, offsets = [3, 1, -1, 4, 1], [0, N // 3, N // 3 + 20, N // 3 + 25, N - 5, N]                  # (rising: N > 45)
    for P, Q in ((A1.expand(r, K, n), B), (A, B1.expand(M, r, n)), (A1.expand(r, K, n), B1.expand(M, r, n))):
        y, back = nb.adapter_mul_pullback(W, X, P, Q, _ints(ids), offsets=_ints(offsets))
        w, x, p, q, d, s = _f64(W), _f64(X), _f64(P), _f64(Q), _f64(dY), np.ones(n)
        sizes = _sizes(w, x, p, q, ids, offsets, s, dtype, d)
        _close(y, R.adapters(w, x, p, q, ids, offsets, s), dtype, sizes[0], "Y")
        for got, want, size, what in zip(back(dY), R.adapters_back(w, x, p, q, ids, offsets, s, d), sizes[1:], ("dX", "dA", "dB")):
            _close(got, want, dtype, size, what)


def _same_kind(got, want, base, others, near, size, dtype, what):
    """NaN and the infinities where the definition has them; in columns of other requests the bits of a call without them, in the pair's own rows without
    them what the definition gives (near: with zeros in their place)."""
    assert (got[:, others] == base[:, others]).all(), what
    got = _f64(got)
    assert (np.isnan(got) == np.isnan(want)).all(), what
    for s in (np.inf, -np.inf):
        assert ((got == s) == (want == s)).all(), what
    fine = np.isfinite(want)
    _close(torch.from_numpy(np.where(fine, got, near)), near, dtype, size, what)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("turn", [(0, 0, 0), (1, 1, 1)])
@pytest.mark.parametrize("M,K,r,lens", [
    (136, 64, 16, [10, 50, 1, 39, 50, 17, 33]), (100, 200, 40, [7, 9, 20]), (512, 328, 16, [300, 5, 129, 64, 20, 240, 1]),
    (320, 136, 100, [64, 32, 16, 500, 3, 40, 200]), (264, 1024, 8, [1] * 24), (512, 200, 64, [512, 256, 256]), (300, 72, 5, [31, 33, 600]), (136, 64, 8, [1] * 900)])
def test_a_pair_with_infinities_reaches_its_own_columns_alone(dtype, turn, M, K, r, lens):
    """Whatever the other requests of a tile are; the pullback's dX is the same product."""
    gen = np.random.default_rng(M + K)
    n = 6
    W, A, B = _factors(gen, M, K, r, n, dtype, turn)
    N = sum(lens)
    X, dY = _cols(gen.standard_normal((K, N)), dtype), _cols(gen.standard_normal((M, N)), dtype)
    ids, offsets = [(2, 0, 5, 1, -1, 3)[i % 6] for i in range(len(lens))], np.concatenate(([0], np.cumsum(lens))).astype(int)
    how = {"offsets": _ints(offsets)}
    run = lambda: (lambda y, back: (y, *back(dY)))(*nb.adapter_mul_pullback(W, X, A, B, _ints(ids), **how))
    base = run()
    inf = float("inf")
    B[M // 2, r // 2, 0], B[3, 0, 5], B[min(M - 1, 70), r - 1, 5] = inf, float("nan"), -inf
    B[M - 1, 0, 2], B[M - 1, r - 1, 2] = inf, inf
    got = run()
    w, x, a, b, d, s = _f64(W), _f64(X), _f64(A), _f64(B), _f64(dY), np.ones(n)
    others = [i for (p, q), e in zip(R.runs(offsets, N), ids) if e in (1, 3, -1) for i in range(p, q)]
    zeros = lambda v: np.where(np.isfinite(v), v, 0.0)
    with np.errstate(invalid="ignore"):
        _same_kind(got[0], R.adapters(w, x, a, b, ids, offsets, s), base[0], others, R.adapters(w, x, a, zeros(b), ids, offsets, s),
                   _sizes(w, x, a, zeros(b), ids, offsets, s, dtype), dtype, "Y")
    B[:] = _cols(np.where(np.isfinite(b), b, 0.25), dtype)
    base = run()
    A[0, K // 2, 0], A[r - 1, K - 1, 5], A[r // 2, 0, 5] = inf, float("nan"), -inf
    got = run()
    a, b = _f64(A), _f64(B)
    others = [i for (p, q), e in zip(R.runs(offsets, N), ids) if e not in (0, 5) for i in range(p, q)]
    with np.errstate(invalid="ignore"):
        _same_kind(got[1], R.adapters_back(w, x, a, b, ids, offsets, s, d)[0], base[1], others, R.adapters_back(w, x, zeros(a), b, ids, offsets, s, d)[0],
                   _sizes(w, x, zeros(a), b, ids, offsets, s, dtype, d)[1], dtype, "dX")
    assert (got[2] == base[2]).all()                         # (dA = scale B^T dY X^T)


@pytest.mark.gpu
@pytest.mark.parametrize("turn", [(0, 0, 0), (1, 1, 1)])
@pytest.mark.parametrize("M,K,r,lens", [(256, 136, 16, [300, 300]), (264, 200, 48, [700, 3, 500]), (130, 72, 100, [2000]), (128, 1024, 8, [1] * 40), (64, 33, 16, [9000])])
def test_gradients_of_small_float16_numbers(turn, M, K, r, lens):
    """scale * B^T dY of a training step is of some 1e-6, and scale * A X of small columns too: what is kept of them may not be what the gradients are off by.
    Two Float16 terms, the second 2^11 times as large: |T| * 2^-22, and 2^-36, half a step of Float16's smallest numbers (2^-25) / 2^11."""
    gen = np.random.default_rng(M + r)
    N, n = sum(lens), 3
    offsets, ids = np.concatenate(([0], np.cumsum(lens))).astype(int), [i % n for i in range(len(lens))]
    W, A, B = _factors(gen, M, K, r, n, F16, turn)
    w, a, b, s = _f64(W), _f64(A), _f64(B), np.full(n, 0.5)
    for of_x, of_d in ((1.0, 1e-6), (1e-6, 1.0), (1.0, 2e-5)):
        X, dY = _cols(of_x * gen.standard_normal((K, N)), F16), _cols(of_d * gen.standard_normal((M, N)), F16)
        y, back = nb.adapter_mul_pullback(W, X, A, B, _ints(ids), offsets=_ints(offsets), scale=0.5)
        x, d = _f64(X), _f64(dY)
        _close(y, R.adapters(w, x, a, b, ids, offsets, s), F16, _sizes(w, x, a, b, ids, offsets, s, F16), "Y")
        dX, dA, dB = R.adapters_back(*(np.abs(v) for v in (w, x, a, b)), ids, offsets, s, np.abs(d))
        kept, u = 2.0 ** -22 * 1.01, 2.0 ** -23
        sA, sB = ((N + M + r + 4) * u * 2 + kept) * dA, ((N + K + r + 4) * u * 2 + kept) * dB
        for (p, q), i in zip(R.runs(offsets, N), ids):
            sA[:, :, i] += 2.0 ** -36 * np.abs(x[:, p:q]).sum(1)
            sB[:, :, i] += 2.0 ** -36 * np.abs(d[:, p:q]).sum(1, keepdims=True)
        want = R.adapters_back(w, x, a, b, ids, offsets, s, d)
        got = back(dY)
        _close(got[0], want[0], F16, _sizes(w, x, a, b, ids, offsets, s, F16, d)[1], "dX")
        _close(got[1], want[1], F16, sA, "dA")
        _close(got[2], want[2], F16, sB, "dB")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("N", [40, 200, 1500])
def test_offsets_of_requests_that_fall(dtype, N):
    gen = np.random.default_rng(N)
    M, K, r, n = 264, 136, 16, 4
    W, A, B = _factors(gen, M, K, r, n, dtype)
    X, dY = _cols(gen.standard_normal((K, N)), dtype), _cols(gen.standard_normal((M, N)), dtype)
    w, x, a, b, d, s = _f64(W), _f64(X), _f64(A), _f64(B), _f64(dY), np.ones(n)
    for o in ([1.0, 0.0, 0.4, 0.9, 0.8], [0.9, 0.2, 0.5, 0.5, 0.9], [0.6, 0.9, 0.1, 0.3, 0.0], [0.5, 9.0, 0.1, 0.4, -1.0], [0.8, 0.6, 0.4, 0.2, 0.0]):
        offsets, ids = [int(round(v * N)) for v in o], [1, 3, 0, 2]
        y, back = nb.adapter_mul_pullback(W, X, A, B, _ints(ids), offsets=_ints(offsets))
        sizes = _sizes(w, x, a, b, ids, offsets, s, dtype, d)
        _close(y, R.adapters(w, x, a, b, ids, offsets, s), dtype, sizes[0], o)
        for got, want, size, what in zip(back(dY), R.adapters_back(w, x, a, b, ids, offsets, s, d), sizes[1:], ("dX", "dA", "dB")):
            _close(got, want, dtype, size, (what, o))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("runs,L", [(3001, 1), (700, 3)])
def test_many_requests_of_a_few_columns(dtype, given, runs, L):
    """More than a block looks at in one go, and more columns than are taken one by one."""
    gen = np.random.default_rng(runs)
    M, K, r, n, N = 200, 72, 12, 30, runs * L
    W, A, B = _factors(gen, M, K, r, n, dtype)
    X, ids = _cols(gen.standard_normal((K, N)), dtype), gen.integers(-1, n + 1, runs)
    if given:
        offsets = np.minimum(np.arange(runs + 1) * L + gen.integers(0, L + 1, runs + 1), N)
        y = nb.adapter_mul(W, X, A, B, _ints(ids), offsets=_ints(offsets))
    else:
        offsets = np.arange(runs + 1) * L
        y = nb.adapter_mul(W, nb.jl_reshape(X, (K, L, runs)) if L > 1 else X, A, B, _ints(ids))
        y = nb.jl_reshape(y, (M, N))
    w, x, a, b, s = _f64(W), _f64(X), _f64(A), _f64(B), np.ones(n)
    _close(y, R.adapters(w, x, a, b, ids, offsets, s), dtype, _sizes(w, x, a, b, ids, offsets, s, dtype), "Y")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("turn", [(0, 0, 0), (1, 1, 1)])
@pytest.mark.parametrize("M,K,r,lens", [(136, 72, 8, [200, 90, 300]), (256, 200, 64, [600, 40, 7]), (130, 264, 16, [4000, 3, 700])])
def test_gradients_of_infinite_columns_are_infinite(dtype, turn, M, K, r, lens):
    """An infinity of X or of dY is one of its pair's gradients, of the sign of what it meets, and no NaN unless it meets a zero or another's sign."""
    gen = np.random.default_rng(M + r)
    n, N = 4, sum(lens)
    W, A, B = _factors(gen, M, K, r, n, dtype, turn)
    ids, offsets = [1, 3, 0], np.concatenate(([0], np.cumsum(lens))).astype(int)
    X, dY = _cols(gen.standard_normal((K, N)), dtype), _cols(gen.standard_normal((M, N)), dtype)
    a, b, s = _f64(A), _f64(B), np.full(n, 0.5)
    for of_x in (True, False):
        x, d = X.clone(), dY.clone()
        if of_x:
            x[5, 17], x[K - 1, lens[0] + 2], x[5, 30] = float("inf"), -float("inf"), float("inf")
        else:
            d[7, 17], d[M - 1, lens[0] + 2], d[7, 40] = float("inf"), -float("inf"), float("inf")
        dX, dA, dB = nb.adapter_mul_pullback(W, x, A, B, _ints(ids), offsets=_ints(offsets), scale=0.5)[1](d)
        with np.errstate(invalid="ignore"):
            _, wA, wB = R.adapters_back(_f64(W), _f64(x), a, b, ids, offsets, s, _f64(d))
        for got, want, what in ((dA, wA, "dA"), (dB, wB, "dB")):
            got = _f64(got)
            for e in (np.inf, -np.inf):
                assert ((got == e) == (want == e)).all(), (what, of_x)
            assert (np.isnan(got) == np.isnan(want)).all() and np.isinf(want).any(), (what, of_x)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_captured_call_follows_what_the_pairs_hold(dtype):
    """Whether a pair has infinities is found out on every replay, here by two graphs in turn."""
    gen = np.random.default_rng(9)
    M, K, r, n, N = 264, 136, 16, 3, 800
    W, A, B = _factors(gen, M, K, r, n, dtype)
    X, dY = _cols(gen.standard_normal((K, N)), dtype), _cols(gen.standard_normal((M, N)), dtype)
    ids, offsets = _ints([0, 1, 2]), _ints([0, 300, 310, N])
    run = lambda: (lambda y, back: (y, *back(dY)))(*nb.adapter_mul_pullback(W, X, A, B, ids, offsets=offsets))
    clean, graphs, outs = run(), [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    was = B[5, 3, 1].clone()
    for value in (was, torch.full_like(was, float("inf")), was):
        B[5, 3, 1] = value
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = run()
        for out in outs:
            for a, b, c in zip(out, want, clean):
                assert torch.equal(torch.nan_to_num(a, 7.0, 8.0, 9.0), torch.nan_to_num(b, 7.0, 8.0, 9.0))
                assert value.isinf() or (a == c).all()
        assert value.isfinite() or (torch.isinf(outs[0][0][5, 300:310]).all() and torch.isfinite(outs[0][0][:, :300]).all())
    nb.device_health(DEV)
