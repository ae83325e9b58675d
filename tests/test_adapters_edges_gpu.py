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
