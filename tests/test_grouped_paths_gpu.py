"""Ragged products and adapters at the sizes where another kernel, or another way through one, takes them: pairs of thread blocks on
a tile, K cut into parts, single columns, more runs than a block's table holds, copies of what cannot be addressed.  Tolerances as in
test_experts_gpu.py and test_adapters_gpu.py."""
import numpy as np
import pytest
import torch

import nnlib_jl_b200 as nb
from nnlib_jl_b200 import _lib
from oracle import experts_oracle as R
from test_adapters_gpu import _sizes, _turned
from test_experts_gpu import BF16, DEV, F16, F32, _bound, _close, _cols, _f64, _ints, _matrices

SIXTEEN = [BF16, F16]


def _grouped64(A, X, o, columns=None):
    """R.grouped, a matrix product a run."""
    out = np.zeros((A.shape[0], X.shape[1] if columns is None else len(columns)))
    for g, (a, b) in enumerate(R.runs(o, out.shape[1])):
        out[:, a:b] = A[:, :, g] @ X[:, np.arange(a, b) if columns is None else columns[a:b]]
    return out


def _grad64(dC, X, o, G):
    return np.stack([dC[:, a:b] @ X[:, a:b].T for a, b in R.runs(o, X.shape[1])], 2) if G else None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", SIXTEEN)
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("M,K,G,N", [(1024, 320, 3, 4100), (900, 136, 9, 5001), (300, 1000, 2, 3333), (257, 200, 1, 9000)])
def test_large_tiles_of_ragged_runs(dtype, turned, M, K, G, N):
    gen = np.random.default_rng(M + G)
    o = np.concatenate(([0], np.sort(gen.integers(0, N, G - 1)), [N])).astype(int) if G > 1 else np.array([0, N])
    if G > 2:
        o[1] = o[2]                                          # an empty run
    A, X, dC = _matrices(gen, M, K, G, dtype, turned), _cols(gen.standard_normal((K, N)), dtype), _cols(gen.standard_normal((M, N)), dtype)
    out, back = nb.grouped_mul_pullback(A, X, _ints(o))
    dA, dX = back(dC)
    a, x, d = _f64(A), _f64(X), _f64(dC)
    _close(out, _grouped64(a, x, o), dtype, _bound(K, dtype) * _grouped64(np.abs(a), np.abs(x), o), "C")
    _close(dA, _grad64(d, x, o, G), dtype, _bound(N, dtype) * _grad64(np.abs(d), np.abs(x), o, G), "dA")
    at = a.transpose(1, 0, 2)
    _close(dX, _grouped64(at, d, o), dtype, _bound(M, dtype) * _grouped64(np.abs(at), np.abs(d), o), "dX")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", SIXTEEN)
def test_a_large_run_does_not_see_its_neighbours(dtype):
    gen = np.random.default_rng(2)
    M, K, G, N = 512, 256, 3, 3000
    A, X, dC = _matrices(gen, M, K, G, dtype, False), _cols(gen.standard_normal((K, N)), dtype), _cols(gen.standard_normal((M, N)), dtype)
    o = _ints([0, 1003, 1990, 3000])
    out, back = nb.grouped_mul_pullback(A, X, o)
    dA, dX = back(dC)
    X2, dC2 = X.clone(), dC.clone()
    X2[:, 1003:1990], dC2[:, 1003:1990] = float("nan"), float("inf")
    out2, back2 = nb.grouped_mul_pullback(A, X2, o)
    dA2, dX2 = back2(dC2)
    for a, b in ((out, out2), (dX, dX2)):
        assert (a[:, :1003] == b[:, :1003]).all() and (a[:, 1990:] == b[:, 1990:]).all()
    assert (dA[:, :, 0] == dA2[:, :, 0]).all() and (dA[:, :, 2] == dA2[:, :, 2]).all() and torch.isnan(dA2[:, :, 1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", SIXTEEN)
@pytest.mark.parametrize("M,K,G,k,N", [(136, 1032, 4, 2, 20), (64, 4096, 8, 2, 33), (257, 2048, 2, 1, 5), (40, 777, 3, 2, 50)])
def test_k_in_parts_with_gathered_columns(dtype, M, K, G, k, N):
    gen = np.random.default_rng(K)
    mask = torch.from_numpy(gen.random(N) < 0.8).to(DEV)
    r = nb.route_topk(_cols(gen.standard_normal((G, N))), k, mask=mask)
    A, X = _matrices(gen, M, K, G, dtype, K % 2 == 0), _cols(gen.standard_normal((K, N)), dtype)
    a, x, o, c = _f64(A), _f64(X), r.offsets.cpu().numpy(), r.columns.cpu().numpy()
    want, size = R.grouped(a, x, o, c), _bound(K, dtype) * R.grouped(np.abs(a), np.abs(x), o, c)
    _close(nb.grouped_mul(A, X, r), want, dtype, size)
    keep = _cols(np.full((M, k * N), 3.0), dtype)
    nb.grouped_mul_(keep, A, X, r)
    last = int(o[-1])
    assert (keep[:, last:] == 3).all()
    _close(keep[:, :last], want[:, :last], dtype, size[:, :last])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_more_runs_than_a_table_holds(dtype):
    gen = np.random.default_rng(3)
    M, K, G, N = 24, 40, 1300, 2000
    o = np.sort(gen.integers(0, N + 1, G + 1))
    A, X, dC = _matrices(gen, M, K, G, dtype, False), _cols(gen.standard_normal((K, N)), dtype), _cols(gen.standard_normal((M, N)), dtype)
    out, back = nb.grouped_mul_pullback(A, X, _ints(o))
    dA, dX = back(dC)
    a, x, d = _f64(A), _f64(X), _f64(dC)
    _close(out, _grouped64(a, x, o), dtype, _bound(K, dtype) * _grouped64(np.abs(a), np.abs(x), o))
    _close(dA, _grad64(d, x, o, G), dtype, _bound(N, dtype) * _grad64(np.abs(d), np.abs(x), o, G))


@pytest.mark.gpu
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("M,K,G,N", [(300, 1200, 20, 40), (127, 1027, 9, 30), (64, 2500, 3, 4), (1030, 65, 50, 70), (5, 3000, 2, 5), (512, 640, 6, 300)])
def test_a_few_columns_to_a_run_in_float32(M, K, G, N, turned):
    gen = np.random.default_rng(M + K)
    A, X = _matrices(gen, M, K, G, F32, turned), _cols(gen.standard_normal((K, 17)))
    o = np.sort(gen.integers(0, N + 1, G + 1))
    c = gen.integers(0, 17, N)
    c[N // 2] = 99                                           # no column
    X[:, 5] = float("inf")
    none = torch.empty(0, device=DEV)
    r = nb.Routing(none, none, _ints(o), _ints(c), none)
    a, x = _f64(A), _f64(X)
    fine = np.flatnonzero(c != 5)
    x[:, 5] = 0
    want, size = R.grouped(a, x, o, c), _bound(K, F32) * R.grouped(np.abs(a), np.abs(x), o, c)
    for run in range(2):
        got = nb.grouped_mul(A, X, r) if run else nb.grouped_mul_(_cols(np.full((M, N), 3.0)), A, X, r)
        keep = fine if run else fine[(fine >= o[0]) & (fine < o[-1])]
        _close(got[:, _ints(keep).long()], want[:, keep], F32, size[:, keep])
        if not run:
            assert (got[:, :o[0]] == 3).all() and (got[:, o[-1]:] == 3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("turn", [(0, 0, 0), (1, 1, 1)])
@pytest.mark.parametrize("M,K,r,n,N", [(320, 1024, 16, 7, 20), (131, 1500, 5, 3, 9), (512, 5000, 128, 4, 3), (64, 1024, 3, 2, 500), (40, 100, 8, 70, 64)])
def test_single_columns_in_float32(turn, M, K, r, n, N):
    ids = [(5 * i) % (n + 2) - 1 for i in range(N)]
    for given in (False, True):
        _adapter_case(F32, M, K, r, n, np.arange(N + 1), ids, N, turn, given)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", SIXTEEN)
def test_one_matrix_for_every_run(dtype):
    gen = np.random.default_rng(4)
    M, K, G, N = 136, 64, 5, 400
    one = _matrices(gen, M, K, 1, dtype, False)
    X, o = _cols(gen.standard_normal((K, N)), dtype), _ints([0, 100, 100, 250, 390, 400])
    assert (nb.grouped_mul(one.expand(M, K, G), X, o) == nb.grouped_mul(one, X, _ints([0, N]))).all()


def _adapter_case(dtype, M, K, r, n, offsets, ids, N, turn=(0, 0, 0), given=True, grads=True):
    gen = np.random.default_rng(M + K + r)
    W, A, B = (_turned(_cols(gen.standard_normal(s) / np.sqrt(s[1]), dtype), t) for s, t in zip(((M, K), (r, K, n), (M, r, n)), turn))
    X, dY = _cols(gen.standard_normal((K, N)), dtype), _cols(gen.standard_normal((M, N)), dtype)
    scale = gen.uniform(0.5, 2.0, n)
    how = {"scale": _cols(scale)} | ({"offsets": _ints(offsets)} if given else {})
    y, back = nb.adapter_mul_pullback(W, X, A, B, _ints(ids), **how)
    w, x, a, b, d, s = _f64(W), _f64(X), _f64(A), _f64(B), _f64(dY), np.float32(scale).astype(np.float64)
    sizes = _sizes(w, x, a, b, ids, offsets, s, dtype, d)
    _close(y, R.adapters(w, x, a, b, ids, offsets, s), dtype, sizes[0], "Y")
    if grads:
        for got, want, size, what in zip(back(dY), R.adapters_back(w, x, a, b, ids, offsets, s, d), sizes[1:], ("dX", "dA", "dB")):
            _close(got, want, dtype, size, what)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", SIXTEEN)
@pytest.mark.parametrize("turn", [(0, 0, 0), (1, 1, 1)])
@pytest.mark.parametrize("r", [16, 40, 64, 100])
def test_pairs_that_change_inside_a_large_tile(dtype, turn, r):
    lens = [300, 1, 700, 64, 0, 935, 1000, 17, 500]
    _adapter_case(dtype, 768, 200, r, 5, np.concatenate(([0], np.cumsum(lens))), [0, 1, 2, 2, 3, -1, 4, 0, 4], sum(lens), turn)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", SIXTEEN)
@pytest.mark.parametrize("turn", [(0, 0, 0), (0, 1, 1)])
@pytest.mark.parametrize("M,K,r,n,N", [(320, 1024, 16, 7, 20), (200, 2100, 8, 70, 64), (131, 1500, 5, 3, 9), (512, 5000, 128, 4, 3), (64, 1024, 3, 2, 500), (256, 1030, 48, 2, 31)])
def test_single_columns(dtype, turn, M, K, r, n, N):
    ids = [(5 * i) % (n + 2) - 1 for i in range(N)]
    for given in (False, True):
        _adapter_case(dtype, M, K, r, n, np.arange(N + 1), ids, N, turn, given, grads=given)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", SIXTEEN)
@pytest.mark.parametrize("turn", [(0, 0, 0), (1, 1, 1)])
@pytest.mark.parametrize("M,K,r,n,lens,ids", [(200, 136, 8, 1, [6000], [0]), (130, 264, 40, 1, [1000, 3, 2050, 64, 1900], [0, 0, -1, 0, 0]),
                                              (300, 128, 128, 2, [4000, 10, 5000, 0, 77], [1, 0, 1, 0, 1]), (65, 33, 16, 3, [4500, 4500, 4500], [0, 2, 2])])
def test_gradients_of_few_pairs_and_many_columns(dtype, turn, M, K, r, n, lens, ids):
    _adapter_case(dtype, M, K, r, n, np.concatenate(([0], np.cumsum(lens))), ids, sum(lens), turn)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("given", [False, True])
def test_more_requests_than_a_table_holds(dtype, given):
    gen = np.random.default_rng(5)
    N = 1500
    _adapter_case(dtype, 96, 64, 8, 20, np.arange(N + 1), gen.integers(-1, 20, N), N, given=given)


@pytest.mark.gpu
def test_two_streams_at_once():
    gen = np.random.default_rng(6)
    M, K, G, N = 512, 512, 4, 2000
    A, X = _matrices(gen, M, K, G, BF16, False), [_cols(gen.standard_normal((K, N)), BF16) for _ in range(2)]
    o = [_ints([0, 400, 900, 1500, 2000]), _ints([10, 10, 1000, 1001, 1900])]
    few = [nb.as_column_major(x[:, :40]) for x in X]
    W, P, Q = (_cols(gen.standard_normal(s) / 16, BF16) for s in ((M, K), (16, K, 8), (M, 16, 8)))
    ids = _ints(gen.integers(-1, 8, 40))
    want = [(nb.grouped_mul(A, x, p), nb.adapter_mul(W, f, P, Q, ids)) for x, p, f in zip(X, o, few)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((nb.grouped_mul(A, X[i], o[i]), nb.adapter_mul(W, few[i], P, Q, ids)))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for a, b in g:
            assert (a == w[0]).all() and (b == w[1]).all()
    nb.device_health(DEV)


@pytest.mark.gpu
def test_the_same_call_gives_the_same_bits():
    gen = np.random.default_rng(7)
    M, K, G, N = 384, 256, 6, 1500
    A, X, dC = _matrices(gen, M, K, G, F16, True), _cols(gen.standard_normal((K, N)), F16), _cols(gen.standard_normal((M, N)), F16)
    o = _ints([0, 1, 600, 600, 901, 1400, 1500])
    first = None
    for _ in range(4):
        out, back = nb.grouped_mul_pullback(A, X, o)
        now = (out, *back(dC))
        if first is not None:
            assert all((a == b).all() for a, b in zip(first, now))
        first = now


@pytest.mark.gpu
def test_a_workspace_that_is_too_small_is_refused():
    """An odd leading dimension is copied to one that the copy engine can address: the library says how much that takes."""
    import ctypes as C
    A, X = nb.jl_zeros((33, 35, 2), BF16, DEV), nb.jl_zeros((35, 10), BF16, DEV)
    out, o = nb.jl_zeros((33, 10), BF16, DEV), _ints([0, 5, 10])
    p = _lib.GroupedParams(dtype=_lib.BF16, M=33, K=35, G=2, N=10, R=10, A=A.data_ptr(), lda=33, strideA=33 * 35, X=X.data_ptr(), ldx=35, C=out.data_ptr(),
                           ldc=33, offsets=o.data_ptr())
    lib = _lib.load()
    need = lib.nnlib_b200_grouped_gemm_workspace_bytes(C.byref(p))
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    assert need >= 2 * 40 * 35 * 2 and lib.nnlib_b200_grouped_gemm(C.byref(p), ws.data_ptr(), need - 1, stream) == _lib.WORKSPACE_TOO_SMALL
    assert lib.nnlib_b200_grouped_gemm(C.byref(p), None, 0, stream) == _lib.WORKSPACE_TOO_SMALL
    assert lib.nnlib_b200_grouped_gemm(C.byref(p), ws.data_ptr(), need, stream) == _lib.OK
