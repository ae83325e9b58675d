"""Calls of grouped products that their documentation allows and that went wrong once: a routing of which some experts are held, a
routing of other tokens, one matrix for every run that has to be copied, offsets that fall, a column's place in its tile.  Tolerances as in test_experts_gpu.py."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import nnlib_jl_b200 as nb
from oracle import experts_oracle as R
from test_experts_gpu import BF16, DEV, F16, F32, _bound, _close, _cols, _f64, _ints, _matrices


def _poison(n):
    """What the allocator gives out next is full of NaN."""
    junk = [torch.full((n,), float("nan"), device=DEV) for _ in range(3)]
    torch.cuda.synchronize()
    del junk


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_gathered_gradients_where_some_of_the_experts_are_held(dtype):
    """A part of the offsets, and the matrices of that part: pairs of other experts add nothing to the columns' gradient."""
    gen = np.random.default_rng(1)
    M, K, G, k, N = 72, 136, 6, 3, 100
    r = nb.route_topk(_cols(gen.standard_normal((G, N))), k)
    held = r._replace(offsets=r.offsets[2:5])
    o, c = held.offsets.cpu().numpy(), r.columns.cpu().numpy()
    A, X, dC = _matrices(gen, M, K, 2, dtype, False), _cols(gen.standard_normal((K, N)), dtype), _cols(gen.standard_normal((M, k * N)), dtype)
    out, back = nb.grouped_mul_pullback(A, X, held)
    _poison(K * k * N // 2 if dtype != F32 else K * k * N)
    dA, dX = back(dC)
    a, x, d = _f64(A), _f64(X), _f64(dC)
    wA, wX = R.grouped_back(a, x, o, d, c)
    sA, sX = R.grouped_back(np.abs(a), np.abs(x), o, np.abs(d), c)
    _close(out, R.grouped(a, x, o, c), dtype, _bound(K, dtype) * R.grouped(np.abs(a), np.abs(x), o, c), "C")
    _close(dA, wA, dtype, _bound(k * N, dtype) * sA, "dA")
    _close(dX, wX, dtype, (_bound(M, dtype) + torch.finfo(dtype).eps / 2 * 1.01) * sX + (k * 2.0 ** -25 if dtype == F16 else 0), "dX")


@pytest.mark.gpu
def test_a_routing_of_other_tokens_has_no_gradient():
    r = nb.route_topk(nb.jl_zeros((4, 10), F32, DEV), 2)
    A = nb.jl_zeros((8, 16, 4), F32, DEV)
    for N in (9, 11):
        with pytest.raises(nb.ArgumentError):
            nb.grouped_mul_pullback(A, nb.jl_zeros((16, N), F32, DEV), r)
    with pytest.raises(TypeError):
        nb.grouped_mul_pullback(A, nb.jl_zeros((16, 10), F32, DEV), r._replace(position=r.position.long()))
    nb.grouped_mul_pullback(A, nb.jl_zeros((16, 10), F32, DEV), r)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gathered_arrays_without_features(dtype):
    r = nb.route_topk(nb.jl_zeros((4, 10), F32, DEV), 2)
    for M, K in ((8, 0), (0, 8), (0, 0)):
        out, back = nb.grouped_mul_pullback(nb.jl_zeros((M, K, 4), dtype, DEV), nb.jl_zeros((K, 10), dtype, DEV), r)
        dA, dX = back(nb.jl_zeros((M, 20), dtype, DEV))
        assert tuple(out.shape) == (M, 20) and tuple(dA.shape) == (M, K, 4) and tuple(dX.shape) == (K, 10)
        assert (out == 0).all() and (dX == 0).all()
    y, back = nb.combine_pullback(nb.jl_zeros((0, 20), dtype, DEV), r)
    dY, dw = back(nb.jl_zeros((0, 10), dtype, DEV))
    assert tuple(y.shape) == (0, 10) and tuple(dY.shape) == (0, 20) and (dw == 0).all() and tuple(dw.shape) == (2, 10)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("M,K", [(137, 64), (136, 67), (137, 67)])
def test_one_matrix_for_every_run_that_is_copied(dtype, turned, M, K):
    """The first run is empty: the one copy of the matrix is not its alone."""
    gen = np.random.default_rng(M + K)
    G, N = 5, 400
    one = _matrices(gen, M, K, 1, dtype, turned)
    X, dC, o = _cols(gen.standard_normal((K, N)), dtype), _cols(gen.standard_normal((M, N)), dtype), _ints([0, 0, 100, 250, 390, 400])
    each = _matrices(gen, M, K, G, dtype, turned).copy_(one.expand(M, K, G))
    want = nb.grouped_mul(each, X, o)
    dA, dX = nb.grouped_mul_pullback(each, X, o)[1](dC)
    _poison(M * K * G)
    out, back = nb.grouped_mul_pullback(one.expand(M, K, G), X, o)
    assert (out == want).all()
    _poison(M * K * G)
    gA, gX = back(dC)
    assert (gX == dX).all() and (gA == dA).all()
    few = _ints([0, 0, 3, 5, 9, 12])                        # (gathered, K in parts)
    c = _ints(gen.integers(0, N, 12))
    none = torch.empty(0, device=DEV)
    r = nb.Routing(none, none, few, c, none)
    want = nb.grouped_mul(each, X, r)
    _poison(M * K * G)
    assert (nb.grouped_mul(one.expand(M, K, G), X, r) == want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("M,K,N", [(136, 64, 400), (300, 1000, 70), (72, 333, 40), (520, 130, 20), (264, 96, 9), (96, 70, 3)])
def test_a_columns_result_does_not_depend_on_its_place(M, K, N, turned):
    """Bit by bit, in Float32, whatever the tile: the parts of a sum are added in one order."""
    gen = np.random.default_rng(M + N)
    A, X = _matrices(gen, M, K, 1, F32, turned), _cols(gen.standard_normal((K, N)))
    out = nb.grouped_mul(A, X, _ints([0, N]))
    for by in (1, 2, 5, 8, 19):
        moved = nb.grouped_mul(A, nb.as_column_major(torch.roll(X, by, 1)), _ints([0, N]))
        assert (moved == torch.roll(out, by, 1)).all(), by


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,K,G,N", [(136, 72, 4, 90), (512, 256, 4, 900), (40, 2048, 4, 30), (264, 64, 4, 5000)])
def test_offsets_that_fall(dtype, M, K, G, N):
    """A run that ends before it begins is empty; what no other run has becomes zeros, and nothing else does."""
    gen = np.random.default_rng(M + N)
    A, X, dC = _matrices(gen, M, K, G, dtype, False), _cols(gen.standard_normal((K, N)), dtype), _cols(gen.standard_normal((M, N)), dtype)
    a, x, d = _f64(A), _f64(X), _f64(dC)
    u = lambda v: int(round(v * N))
    for o in ([1.0, 0.0, 0.4, 0.9, 0.8], [0.9, 0.2, 0.5, 0.5, 0.9], [0.6, 0.9, 0.1, 0.3, 0.0], [0.0, 0.5, -3.0, 0.0, 0.0], [0.5, 9.0, 0.1, 0.4, -1.0], [0.8, 0.6, 0.4, 0.2, 0.0]):
        o = [u(v) for v in o]
        out, back = nb.grouped_mul_pullback(A, X, _ints(o))
        want, size = R.grouped(a, x, o), _bound(K, dtype) * R.grouped(np.abs(a), np.abs(x), o)
        _close(out, want, dtype, size, o)
        dA, dX = back(dC)
        wA, wX = R.grouped_back(a, x, o, d)
        sA, sX = R.grouped_back(np.abs(a), np.abs(x), o, np.abs(d))
        _close(dA, wA, dtype, _bound(N, dtype) * sA, o)
        _close(dX, wX, dtype, _bound(M, dtype) * sX, o)
        keep = _cols(np.full((M, N), 7.0), dtype)
        nb.grouped_mul_(keep, A, X, _ints(o))
        want = R.grouped(a, x, o, rest=7.0)
        _close(keep, want, dtype, size, o)


@pytest.mark.gpu
def test_the_log_names_the_way_of_every_product_and_gradient():
    code = ("import torch, nnlib_jl_b200 as nb\n"
            "for t in (torch.bfloat16, torch.float32):\n"
            "    z = lambda *s: nb.jl_zeros(s, t, torch.device('cuda:0'))\n"
            "    i = lambda *v: torch.tensor(v, dtype=torch.int32, device='cuda')\n"
            "    out, back = nb.grouped_mul_pullback(z(64, 32, 2), z(32, 40), i(0, 20, 40)); back(out)\n"
            "    y, back = nb.adapter_mul_pullback(z(64, 32), z(32, 40), z(8, 32, 2), z(64, 8, 2), i(0, 1), offsets=i(0, 20, 40)); back(y)\n")
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, NNLIB_B200_LOG="1", NNLIB_B200_FORCE_SIMT="0"), capture_output=True, text=True)
    lines = [(l.split()[1], l.split("->")[1].strip()) for l in r.stderr.splitlines() if l.startswith("[nnlib_b200]")]
    calls = ["grouped_gemm", "grouped_gemm_grad", "grouped_gemm", "adapter_gemm", "adapter_bwd"]
    assert lines == [(c, way) for way in ("tcgen05", "cuda-core") for c in calls], r.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_matrices_of_one_column_of_wider_ones(dtype):
    gen = np.random.default_rng(8)
    for M in (40, 137, 1):
        A, X, dC = _matrices(gen, M, 9, 3, dtype, True)[:, 3:4], _cols(gen.standard_normal((1, 50)), dtype), _cols(gen.standard_normal((M, 50)), dtype)
        o = [0, 20, 20, 50]
        out, back = nb.grouped_mul_pullback(A, X, _ints(o))
        dA, dX = back(dC)
        a, x, d = _f64(A), _f64(X), _f64(dC)
        _close(out, R.grouped(a, x, o), dtype, _bound(1, dtype) * R.grouped(np.abs(a), np.abs(x), o))
        (wA, wX), (sA, sX) = R.grouped_back(a, x, o, d), R.grouped_back(np.abs(a), np.abs(x), o, np.abs(d))
        _close(dA, wA, dtype, _bound(50, dtype) * sA)
        _close(dX, wX, dtype, _bound(M, dtype) * sX)
