"""Router, grouped products and weighted sums against the Float64 oracle.

Tolerances.  A result is rounded once: half a step of its type, relative to it (Float16 below its normal numbers: 2^-25).  A sum of n products in Float32
before that is off by at most n roundings of 2^-24 of the sum of magnitudes, one for each addition, whatever their order; the tensor
cores cut instead of rounding, which doubles it.  Softmax weights: exponentials of at most 2 units of 2^-23 where the
difference of two Float32 logits is exact or off by 2^-24 of it (|difference| < 16 here: 2^-20 relative in the exponential), a sum of at most 1024 of them and a
division: 2^-19 relative.  Whole numbers are equal."""
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


def _close(got, want, dtype, size, what=""):
    """size: how far Float32 sums may be off"""
    got = _f64(got)
    lim = torch.finfo(dtype).eps / 2 * 1.001 * np.abs(want) + size + (2.0 ** -25 if dtype == F16 else 2.0 ** -126)
    assert got.shape == want.shape and np.isfinite(got).all(), what
    assert (np.abs(got - want) <= lim).all(), (what, float((np.abs(got - want) - lim).max()))


# ------------------------------------------------------------------------------------------------- router
ROUTES = [
    # G, k, N
    (1, 1, 3), (2, 1, 1), (8, 2, 33), (8, 8, 40), (32, 32, 5), (33, 4, 64), (60, 4, 129), (64, 6, 700), (128, 8, 50), (200, 3, 257),
    (256, 8, 1000), (512, 10, 300), (1000, 7, 140), (1024, 32, 20), (5, 2, 0), (4, 2, 9000),
]


def _check_route(logits, k, r, dtype, **how):
    x = _f64(logits)
    bias = how.get("bias")
    mask = how.get("mask")
    w, e, o, c, p = R.route(x, k, None if bias is None else bias.cpu().numpy(), None if mask is None else mask.cpu().numpy(), how.get("normalize", True))
    for got, want in ((r.experts, e), (r.offsets, o), (r.columns, c), (r.position, p)):
        assert got.dtype == torch.int32 and (got.cpu().numpy() == want).all()
    got = _f64(r.weights)
    assert (np.isnan(got) == np.isnan(w)).all()
    there = ~np.isnan(w)
    assert (np.abs(got - w)[there] <= 2.0 ** -19 * w[there] + 2.0 ** -126).all()
    return w, e


@pytest.mark.gpu
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("G,k,N", ROUTES)
def test_route_and_its_pullback(dtype, G, k, N, normalize):
    gen = np.random.default_rng(G + N)
    logits = _cols(gen.standard_normal((G, N)) * 2, dtype)
    if N > 2:
        logits[:, 1] = float(logits[0, 1])               # all equal: the first k
    bias = _cols(gen.standard_normal(G)) if N % 2 else None
    mask = torch.from_numpy(gen.random(N) < 0.8).to(DEV) if N % 3 == 0 else None
    r, back = nb.route_topk_pullback(logits, k, bias=bias, mask=mask, normalize=normalize)
    w, e = _check_route(logits, k, r, dtype, bias=bias, mask=mask, normalize=normalize)
    dw = gen.standard_normal((k, N))
    got = back(_cols(dw))
    want = R.route_back(_f64(logits), e, np.float32(dw).astype(np.float64), normalize)
    # w (dw - sum w dw): 2^-19 of w times the largest dw, for each of the terms, and a sum of at most 32
    size = 2.0 ** -16 * np.abs(dw).max(0, initial=0.0) if k else 0.0
    _close(got, want, dtype, np.broadcast_to(size, want.shape), "dlogits")


@pytest.mark.gpu
@pytest.mark.parametrize("normalize", [True, False])
def test_route_of_infinities_and_nan(normalize):
    inf, nan = np.inf, np.nan
    x = np.array([[0, 1, 2, 3, 4], [-inf, -inf, -inf, 1, -inf], [-inf] * 5, [inf, 0, inf, inf, 1], [nan, 1, 2, -inf, 0],
                  [nan] * 5, [1, -0.0, 0.0, -1, -inf], [inf, nan, 0, 0, 0]]).T
    logits = _cols(x)
    r = nb.route_topk(logits, 3, normalize=normalize)
    _check_route(logits, 3, r, F32, normalize=normalize)
    assert sorted(r.experts[:, 2].tolist()) == [0, 1, 2]      # nothing to choose by: still experts that there are


@pytest.mark.gpu
def test_route_of_strided_logits_and_a_batch_of_ended_sequences():
    gen = np.random.default_rng(5)
    wide = _cols(gen.standard_normal((40, 90)))
    logits = wide[3:35]
    _check_route(logits, 4, nb.route_topk(logits, 4), F32)
    none = torch.zeros(90, dtype=torch.bool, device=DEV)
    r = nb.route_topk(logits, 4, mask=none)
    assert (r.offsets == 0).all() and (r.columns == -1).all() and (r.position == -1).all() and (r.weights == 0).all()


# ------------------------------------------------------------------------------------------------- products
def _offsets(gen, G, N, how="random"):
    if how == "one":                                         # all in the last group
        return np.array([0] * G + [N])
    if how == "gap":                                         # columns before the first and behind the last run
        return np.sort(gen.integers(N // 5, max(N - N // 5, 1), G + 1))
    cuts = np.sort(gen.integers(0, N + 1, G - 1)) if G > 1 else np.array([], int)
    return np.concatenate(([0], cuts, [N]))


PRODUCTS = [
    # M, K, G, N, offsets
    (128, 64, 4, 200, "random"), (256, 128, 3, 700, "random"), (64, 72, 2, 33, "random"), (40, 8, 5, 17, "gap"), (333, 200, 5, 600, "random"),
    (7, 5, 3, 11, "random"), (1, 1, 2, 3, "random"), (136, 1000, 6, 300, "gap"), (512, 264, 2, 1100, "one"), (264, 520, 40, 90, "random"),
    (1000, 96, 1, 513, "one"), (96, 2048, 16, 16, "random"), (300, 77, 300, 128, "random"), (520, 264, 7, 2000, "gap"), (16, 16, 1, 1, "one"),
]


def _bound(K, dtype):
    return (K + 2) * 2.0 ** (-24 if dtype == F32 else -23)


def _matrices(gen, M, K, G, dtype, turned):
    a = gen.standard_normal((M, K, G)) / np.sqrt(K)
    return _cols(a.transpose(1, 0, 2), dtype).transpose(0, 1) if turned else _cols(a, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,K,G,N,how", PRODUCTS)
def test_grouped_mul_and_its_pullback(dtype, M, K, G, N, how, turned):
    gen = np.random.default_rng(M + K + N)
    o = _offsets(gen, G, N, how)
    A, X, dC = _matrices(gen, M, K, G, dtype, turned), _cols(gen.standard_normal((K, N)), dtype), _cols(gen.standard_normal((M, N)), dtype)
    out, back = nb.grouped_mul_pullback(A, X, _ints(o))
    dA, dX = back(dC)
    assert dA.stride()[:2] == A.stride()[:2] or 1 in (M, K)
    a, x, d = _f64(A), _f64(X), _f64(dC)
    _close(out, R.grouped(a, x, o), dtype, _bound(K, dtype) * R.grouped(np.abs(a), np.abs(x), o), "C")
    wA, wX = R.grouped_back(a, x, o, d)
    sA, sX = R.grouped_back(np.abs(a), np.abs(x), o, np.abs(d))
    _close(dA, wA, dtype, _bound(N, dtype) * sA, "dA")
    _close(dX, wX, dtype, _bound(M, dtype) * sX, "dX")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,K,G,k,N", [(128, 64, 8, 2, 100), (264, 136, 5, 3, 333), (31, 45, 4, 2, 60), (512, 256, 3, 2, 700), (72, 40, 64, 6, 9)])
def test_gathered_products_and_their_pullback(dtype, M, K, G, k, N):
    gen = np.random.default_rng(M + N)
    mask = torch.from_numpy(gen.random(N) < 0.9).to(DEV)
    r = nb.route_topk(_cols(gen.standard_normal((G, N))), k, mask=mask)
    o, c = r.offsets.cpu().numpy(), r.columns.cpu().numpy()
    A, X, dC = _matrices(gen, M, K, G, dtype, N % 2 == 0), _cols(gen.standard_normal((K, N)), dtype), _cols(gen.standard_normal((M, k * N)), dtype)
    out, back = nb.grouped_mul_pullback(A, X, r)
    dA, dX = back(dC)
    a, x, d = _f64(A), _f64(X), _f64(dC)
    _close(out, R.grouped(a, x, o, c), dtype, _bound(K, dtype) * R.grouped(np.abs(a), np.abs(x), o, c), "C")
    wA, wX = R.grouped_back(a, x, o, d, c)
    sA, sX = R.grouped_back(np.abs(a), np.abs(x), o, np.abs(d), c)
    _close(dA, wA, dtype, _bound(k * N, dtype) * sA, "dA")
    # each of a column's k parts is rounded to the type before they are added
    _close(dX, wX, dtype, (_bound(M, dtype) + torch.finfo(dtype).eps / 2 * 1.01) * sX + (k * 2.0 ** -25 if dtype == F16 else 0), "dX")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_columns_in_no_run_and_offsets_out_of_range(dtype):
    gen = np.random.default_rng(1)
    M, K, G, N = 136, 72, 4, 90
    A, X = _matrices(gen, M, K, G, dtype, False), _cols(gen.standard_normal((K, N)), dtype)
    X[:, 80:] = float("nan")                                 # padding behind the last run
    A[:, :, 2] = float("inf")                                # a matrix that no column meets
    o = np.array([5, 30, 30, 30, 80])
    out = nb.grouped_mul(A, X, _ints(o))
    assert torch.isfinite(out).all() and (out[:, :5] == 0).all() and (out[:, 80:] == 0).all()
    keep = _cols(np.full((M, N), 7.0), dtype)
    nb.grouped_mul_(keep, A, X, _ints(o))
    assert (keep[:, :5] == 7).all() and (keep[:, 80:] == 7).all() and (keep[:, 5:80] == out[:, 5:80]).all()
    for o in ([-3, 30, 20, 60, 1000], [0, 0, 0, 0, 0], [90, 90, 90, 90, 90], [200, 300, 400, 500, 600]):
        X2 = _cols(gen.standard_normal((K, N)), dtype)
        A2 = _matrices(gen, M, K, G, dtype, False)
        if o[1] == 30:
            o = [-3, 30, 30, 60, 1000]
        got = nb.grouped_mul(A2, X2, _ints(o))
        want = R.grouped(_f64(A2), _f64(X2), o)
        _close(got, want, dtype, _bound(K, dtype) * R.grouped(np.abs(_f64(A2)), np.abs(_f64(X2)), o))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_run_does_not_see_its_neighbours(dtype):
    """Tiles reach beyond a run's end: what lies there is another run's, infinities and NaN among it."""
    gen = np.random.default_rng(2)
    M, K, G, N = 200, 136, 3, 400
    A, X, dC = _matrices(gen, M, K, G, dtype, False), _cols(gen.standard_normal((K, N)), dtype), _cols(gen.standard_normal((M, N)), dtype)
    o = _ints([0, 131, 270, 400])
    out, back = nb.grouped_mul_pullback(A, X, o)
    dA, dX = back(dC)
    X2, dC2 = X.clone(), dC.clone()
    X2[:, 131:270], dC2[:, 131:270] = float("nan"), float("inf")
    out2, back2 = nb.grouped_mul_pullback(A, X2, o)
    dA2, dX2 = back2(dC2)
    for a, b in ((out, out2), (dX, dX2)):
        assert (a[:, :131] == b[:, :131]).all() and (a[:, 270:] == b[:, 270:]).all()
    assert (dA[:, :, 0] == dA2[:, :, 0]).all() and (dA[:, :, 2] == dA2[:, :, 2]).all() and torch.isnan(dA2[:, :, 1]).all()


@pytest.mark.gpu
def test_columns_of_no_token():
    gen = np.random.default_rng(3)
    for dtype in (F32, BF16):
        M, K, G, N, n = 64, 40, 2, 30, 50
        c = gen.integers(0, N, n)
        c[[3, 20, 44]] = [-1, N, 10 ** 6]
        o = np.array([0, 25, 50])
        none = torch.empty(0, device=DEV)
        r = nb.Routing(none, none, _ints(o), _ints(c), none)
        A, X = _matrices(gen, M, K, G, dtype, True), _cols(gen.standard_normal((K, N)), dtype)
        got = nb.grouped_mul(A, X, r)
        a, x = _f64(A), _f64(X)
        _close(got, R.grouped(a, x, o, c), dtype, _bound(K, dtype) * R.grouped(np.abs(a), np.abs(x), o, c))
        assert (got[:, [3, 20, 44]] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
def test_views_of_wider_arrays_and_odd_alignment(dtype):
    gen = np.random.default_rng(4)
    G, N = 3, 150
    for M, K, off in ((64, 48, 0), (65, 47, 1), (64, 48, 3), (120, 33, 8)):
        wide_a, wide_x = _cols(gen.standard_normal((M + 9, K, G)) / np.sqrt(K), dtype), _cols(gen.standard_normal((K + 20, N)), dtype)
        A, X = wide_a[off:off + M], wide_x[off:off + K]
        o = _offsets(gen, G, N)
        wide_c = _cols(np.full((M + 9, N), 3.0), dtype)
        Cm = wide_c[off:off + M]
        nb.grouped_mul_(Cm, A, X, _ints(o))
        a, x = _f64(A), _f64(X)
        _close(Cm, R.grouped(a, x, o), dtype, _bound(K, dtype) * R.grouped(np.abs(a), np.abs(x), o))
        assert (wide_c[:off] == 3).all() and (wide_c[off + M:] == 3).all()
        out, back = nb.grouped_mul_pullback(A, X, _ints(o))
        d = wide_c[off:off + M]
        dA, dX = back(d)
        wA, wX = R.grouped_back(a, x, o, _f64(d))
        sA, sX = R.grouped_back(np.abs(a), np.abs(x), o, np.abs(_f64(d)))
        _close(dA, wA, dtype, _bound(N, dtype) * sA)
        _close(dX, wX, dtype, _bound(M, dtype) * sX)


@pytest.mark.gpu
def test_empty_products():
    for dtype in (F32, BF16):
        for M, K, G, N in ((0, 8, 2, 5), (8, 0, 2, 5), (8, 8, 2, 0), (8, 8, 0, 5)):
            A, X = nb.jl_zeros((M, K, G), dtype, DEV), nb.jl_zeros((K, N), dtype, DEV)
            o = torch.zeros(G + 1, dtype=torch.int32, device=DEV)
            out, back = nb.grouped_mul_pullback(A, X, o)
            assert tuple(out.shape) == (M, N) and (out == 0).all()
            dA, dX = back(nb.jl_zeros((M, N), dtype, DEV))
            assert tuple(dA.shape) == (M, K, G) and (dA == 0).all() and tuple(dX.shape) == (K, N) and (dX == 0).all()


# ------------------------------------------------------------------------------------------------- weighted sums
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("E,G,k,N", [(8, 4, 2, 5), (64, 8, 2, 33), (37, 5, 3, 40), (4096, 8, 2, 9), (1000, 16, 6, 21), (1, 2, 1, 3), (512, 32, 32, 4), (16, 3, 2, 0)])
def test_combine_and_its_pullback(dtype, E, G, k, N):
    gen = np.random.default_rng(E + N)
    mask = torch.from_numpy(gen.random(N) < 0.8).to(DEV)
    r = nb.route_topk(_cols(gen.standard_normal((G, N))), k, mask=mask)
    p, w = r.position.cpu().numpy(), _f64(r.weights)
    Y, dy = _cols(gen.standard_normal((E, k * N)), dtype), _cols(gen.standard_normal((E, N)), dtype)
    y, back = nb.combine_pullback(Y, r)
    dY, dw = back(dy)
    Y64, d64 = _f64(Y), _f64(dy)
    eps = 2.0 ** -24
    _close(y, R.combine(Y64, p, w), dtype, (k + 1) * eps * R.combine(np.abs(Y64), p, w), "y")
    wY, ww = R.combine_back(Y64, p, w, d64)
    _, sw = R.combine_back(np.abs(Y64), p, w, np.abs(d64))
    _close(dY, wY, dtype, eps * np.abs(wY), "dY")
    _close(dw, ww, F32, (E + 1) * eps * sw, "dw")
    other = _cols(gen.standard_normal((k, N)))
    _close(nb.combine(Y, r, other), R.combine(Y64, p, _f64(other)), dtype, (k + 1) * eps * R.combine(np.abs(Y64), p, np.abs(_f64(other))), "weights")


@pytest.mark.gpu
def test_combine_of_positions_that_are_not():
    gen = np.random.default_rng(9)
    E, N, k, n = 24, 6, 2, 10
    p = gen.integers(0, n, (k, N))
    p[0, 0], p[1, 2], p[0, 5] = -1, n, 10 ** 9
    w = gen.standard_normal((k, N))
    Y = _cols(gen.standard_normal((E, n)))
    Y[:, 0] = 5.0
    c = np.full(n, -1)
    c[3], c[4] = 0, 10 ** 6                                   # neither names a pair, or any token
    p[:, 0] = -1
    none = torch.empty(0, device=DEV)
    r = nb.Routing(_cols(w), none, none, _ints(c), _ints(p))
    y, back = nb.combine_pullback(Y, r)
    want = R.combine(_f64(Y), p, np.float32(w).astype(np.float64))
    _close(y, want, F32, 4 * 2.0 ** -24 * R.combine(np.abs(_f64(Y)), p, np.abs(w)))
    dY, dw = back(_cols(gen.standard_normal((E, N))))
    assert (dY == 0).all() and (dw == 0).all()


# ------------------------------------------------------------------------------------------------- together
def _layer(x, logits, A1, A2, k):
    r, back_r = nb.route_topk_pullback(logits, k)
    h, back_1 = nb.grouped_mul_pullback(A1, x, r)
    a = torch.relu(h)
    z, back_2 = nb.grouped_mul_pullback(A2, a, r.offsets)
    y, back_c = nb.combine_pullback(z, r)

    def back(dy):
        dz, dw = back_c(dy)
        dA2, da = back_2(dz)
        dA1, dx = back_1(torch.where(h > 0, da, torch.zeros_like(da)))
        return dx, back_r(dw), dA1, dA2

    return y, back


@pytest.mark.gpu
def test_a_layer_of_experts_and_its_gradients_by_differences():
    """The gradients against central differences of the layer's own Float32 results along random directions, taken far from
    other choices of experts: the layer is piecewise smooth, so a step of 2^-7 leaves an error of the third derivative and of
    rounding, together below 1 % for these sizes."""
    gen = np.random.default_rng(7)
    E, F, G, k, N = 24, 40, 6, 2, 50
    x, lg = gen.standard_normal((E, N)), gen.standard_normal((G, N))
    order = np.sort(lg, 0)
    lg[:, (order[-k] - order[-k - 1]) < 0.1] += 3 * np.eye(G)[:, [0, 1]].sum(1, keepdims=True)
    mats = [gen.standard_normal((F, E, G)) / np.sqrt(E), gen.standard_normal((E, F, G)) / np.sqrt(F)]
    args = [_cols(v) for v in (x, lg, *mats)]
    y, back = _layer(*args, k)
    dy = _cols(gen.standard_normal((E, N)))
    grads = back(dy)
    for i, (v, g) in enumerate(zip(args, grads)):
        u = _cols(gen.standard_normal(tuple(v.shape)))
        u = u / u.norm()
        step = 2.0 ** -7
        both = []
        for s in (step, -step):
            moved = list(args)
            moved[i] = nb.as_column_major(v + s * u)
            both.append(float((_layer(*moved, k)[0].double() * dy.double()).sum()))
        want = (both[0] - both[1]) / (2 * step)
        got = float((g.double() * u.double()).sum())
        # relu's kinks: an input within a step of 0 changes slope
        assert abs(got - want) <= 2e-2 * float(g.double().norm()) / np.sqrt(g.numel()) + 1e-2 * abs(want) + 2e-3, (i, got, want)


@pytest.mark.gpu
def test_a_captured_layer_follows_new_logits_and_another_stream():
    gen = np.random.default_rng(8)
    E, F, G, k, N = 64, 128, 8, 2, 96
    x, logits = _cols(gen.standard_normal((E, N)), BF16), _cols(gen.standard_normal((G, N)), BF16)
    A1, A2 = _matrices(gen, F, E, G, BF16, False), _matrices(gen, E, F, G, BF16, True)

    def layer():
        r = nb.route_topk(logits, k)
        return nb.combine(nb.grouped_mul(A2, torch.relu(nb.grouped_mul(A1, x, r)), r.offsets), r)

    layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer()
    torch.cuda.current_stream().wait_stream(side)
    for s in range(3):
        g = np.random.default_rng(s)
        logits.copy_(_cols(g.standard_normal((G, N)) + (10 * np.eye(G)[:, [s]]), BF16))
        x.copy_(_cols(g.standard_normal((E, N)), BF16))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        assert (got == layer()).all()
    nb.device_health(DEV)


@pytest.mark.gpu
def test_refusals():
    A, X, o = nb.jl_zeros((8, 16, 2), F32, DEV), nb.jl_zeros((16, 10), F32, DEV), _ints([0, 5, 10])
    for bad in (lambda: nb.grouped_mul(A.cpu(), X, o), lambda: nb.grouped_mul(A, X.half(), o), lambda: nb.grouped_mul(A, X, o.long()),
                lambda: nb.grouped_mul(A[::2], X, o), lambda: nb.grouped_mul(A, X[::2], o), lambda: nb.grouped_mul(A.double(), X.double(), o),
                lambda: nb.grouped_mul(A, X.unsqueeze(2), o), lambda: nb.route_topk(X.int(), 2), lambda: nb.route_topk(X.cpu(), 2),
                lambda: nb.route_topk(X, 2, mask=torch.ones(10, device=DEV)), lambda: nb.route_topk(X, 2, bias=torch.ones(16, device=DEV).half())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: nb.grouped_mul(A, nb.jl_zeros((8, 10), F32, DEV), o), lambda: nb.grouped_mul(A, X, o[:2]), lambda: nb.route_topk(X, 0),
                lambda: nb.route_topk(X, 17), lambda: nb.route_topk(X, 2, mask=torch.ones(9, dtype=torch.bool, device=DEV)),
                lambda: nb.route_topk(X, 2, bias=torch.ones(3, device=DEV)), lambda: nb.grouped_mul_(nb.jl_zeros((8, 9), F32, DEV), A, X, o)):
        with pytest.raises(nb.ArgumentError):
            bad()
    r = nb.route_topk(X, 2)
    with pytest.raises(nb.ArgumentError):
        nb.combine(nb.jl_zeros((4, 20), F32, DEV), r, nb.jl_zeros((3, 10), F32, DEV))
    with pytest.raises(TypeError):
        nb.combine(nb.jl_zeros((4, 20), F32, DEV), r, nb.jl_zeros((2, 10), F16, DEV))
    with pytest.raises(Exception):
        nb.route_topk(nb.jl_zeros((1025, 3), F32, DEV), 2)
