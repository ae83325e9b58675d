"""Norm and rotation of heads and the pullback against the Float64 oracle.

Tolerances: a result is rounded once (half a step of its type, relative), on top of Float32 arithmetic whose errors are
relative to the size of the row: a sum of at most 256 squares in registers and shuffles (at most 24 roundings in a row), a
division, a square root, two products, sine and cosine (2 units) and two products and a sum: below 2^-18 of the row's largest
element of n for the forward pass.  The pullback has two such sums, 2^-17 of the largest r |w|, and cancels.  dg sums N terms
in Float32, each with the forward pass's relative error, in partial sums of at most a few hundred terms in a row:
2^-15 of the sum of magnitudes."""
import numpy as np
import pytest
import torch

import nnlib_jl_b200 as nb
from oracle import rotary_oracle as R

DEV = torch.device("cuda:0")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _array(gen, shape, dtype):
    return nb.jl_from_numpy(gen.standard_normal(shape).astype(np.float32), device=DEV).to(dtype)


def _f64(t):
    return nb.jl_to_numpy(t.double() if t.dtype == F32 else t).astype(np.float64)


def _positions(L, B, start=0, positions=None):
    if positions is not None:
        p = positions.cpu().numpy().astype(np.float64)
        return p if p.ndim == 2 else np.repeat(p[:, None], B, 1)
    s = start.cpu().numpy() if isinstance(start, torch.Tensor) else np.full(B, start)
    return np.arange(L)[:, None] + s[None].astype(np.float64)


def _close(got, want, dtype, size, what):
    """size: what Float32 errors are relative to, broadcastable"""
    err = np.abs(got - want)
    lim = _half_step(dtype) * np.abs(want) * 1.001 + size + (2.0 ** -25 if dtype == F16 else 0)
    assert np.isfinite(got).all() and (err <= lim).all(), (what, float((err - lim).max()))


def _check(q, k, gq, gk, freqs, H, dyq=None, dyk=None, interleaved=False, eps=1e-6, **how):
    d = gq.shape[0]
    _, L, B = q.shape
    pos = _positions(L, B, **how)
    f = freqs.cpu().numpy()
    if dyq is None:
        y = nb.qk_norm_rope(q, k, gq, gk, freqs, nheads=H, interleaved=interleaved, eps=eps, **how)
        got = None
    else:
        *y, back = nb.qk_norm_rope_pullback(q, k, gq, gk, freqs, nheads=H, interleaved=interleaved, eps=eps, **how)
        got = back(dyq, dyk)
    for n, (x, g, dy) in enumerate(((q, gq, dyq), (k, gk, dyk))):
        x64, g64 = _f64(x), _f64(g)
        want = R.norm_rope(x64, g64, pos, f, eps, interleaved)
        row = np.abs(R.heads(want, d)).max(0, keepdims=True) * np.sqrt(2)
        _close(_f64(y[n]), want, x.dtype, R.unheads(np.broadcast_to(2.0 ** -18 * row, (d, *row.shape[1:]))), "y")
        if dy is None:
            continue
        dx, dg = R.pullback(x64, g64, pos, f, eps, interleaved, _f64(dy))
        xh, dyh = R.heads(x64, d), R.heads(_f64(dy), d)
        r = 1 / np.sqrt((xh * xh).mean(0) + eps)
        w = r * np.abs(dyh).max(0) * np.abs(g64).max() * 2 * np.maximum(1, r * np.abs(xh).max(0))
        _close(_f64(got[n]), dx, x.dtype, R.unheads(np.broadcast_to(2.0 ** -17 * w, (d, *w.shape))), "dx")
        u = R.rotate(dyh, pos, f, interleaved, back=True)
        _close(_f64(got[2 + n]), dg, g.dtype, 2.0 ** -15 * np.abs(u * xh * r).sum((1, 2, 3)), "dg")


CASES = [
    # d, rotated, neighbours, query heads, key heads, L, B
    (128, 128, False, 32, 8, 5, 2),
    (128, 128, True, 4, 4, 9, 1),
    (80, 40, True, 8, 8, 33, 3),
    (80, 40, False, 3, 1, 17, 2),
    (64, 64, False, 12, 12, 1, 1),
    (256, 128, False, 5, 2, 7, 2),
    (256, 256, True, 1, 1, 3, 3),
    (112, 112, False, 6, 3, 40, 2),
    (34, 34, False, 3, 2, 6, 2),          # single pairs: no vector fits
    (254, 20, True, 2, 1, 4, 1),          # four pairs to a lane
    (2, 2, True, 1, 1, 3, 2),
    (48, 0, False, 2, 2, 5, 1),           # norm only
    (128, 64, False, 7, 1, 700, 2),       # several tokens to a block
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", CASES)
def test_forward_and_pullback_match_the_oracle(dtype, case):
    d, rot, inter, H, Hk, L, B = case
    gen = np.random.default_rng(3)
    q, k, dyq, dyk = (_array(gen, (h * d, L, B), dtype) for h in (H, Hk, H, Hk))
    gq, gk = (1 + 0.2 * _array(gen, (d,), F32)).to(dtype), (1 + 0.2 * _array(gen, (d,), F32)).to(dtype)
    _check(q, k, gq, gk, nb.rope_frequencies(rot), H, dyq, dyk, inter, start=7)


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["start", "positions", "shared", "far", "negative"])
def test_positions(how):
    d, H, Hk, L, B = 64, 4, 2, 11, 3
    gen = np.random.default_rng(4)
    q, k = _array(gen, (H * d, L, B), F32), _array(gen, (Hk * d, L, B), F32)
    g = torch.ones(d, device=DEV)
    arg = {"start": {"start": torch.tensor([0, 900, 31], dtype=torch.int32, device=DEV)},
           "positions": {"positions": nb.jl_from_numpy(gen.integers(0, 5000, (L, B)).astype(np.int32), device=DEV)},
           "shared": {"positions": torch.arange(5, 5 + L, dtype=torch.int32, device=DEV)},
           "far": {"start": 2_000_000_000},
           "negative": {"start": -20}}[how]
    _check(q, k, g, g, nb.rope_frequencies(d), H, **arg)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_views_into_one_projection(dtype, shift):
    """q and k as slices of a packed array, at offsets that allow 16-byte, 8-byte and single loads; Float32 weights."""
    d, H, Hk, L, B = 64, 4, 2, 13, 2
    gen = np.random.default_rng(5)
    packed = _array(gen, ((H + 2 * Hk) * d + 8, L, B), dtype)
    q, k = packed[shift:shift + H * d], packed[shift + H * d:shift + (H + Hk) * d]
    assert q.stride() == (1, packed.shape[0], packed.shape[0] * L)
    dy = _array(gen, (H * d + 3, L, B), dtype)[shift // 2:shift // 2 + H * d]
    gq, gk = 1 + 0.2 * _array(gen, (d,), F32), 1 + 0.2 * _array(gen, (d,), F32)
    _check(q, k, gq, gk, nb.rope_frequencies(d), H, dy, _array(gen, (Hk * d, L, B), dtype), start=2)


@pytest.mark.gpu
def test_rows_of_zeros_and_large_and_small_ones():
    d, H, L, B = 32, 2, 4, 1
    gen = np.random.default_rng(6)
    q = _array(gen, (H * d, L, B), F32)
    q[:, 0] = 0
    q[:, 1] *= 1e-12
    q[:, 2] *= 1e12
    dy = _array(gen, (H * d, L, B), F32)
    g = torch.ones(d, device=DEV)
    _check(q, q, g, g, nb.rope_frequencies(d), H, dy, dy, eps=1e-6)
    y, _ = nb.qk_norm_rope(q, q, g, g, nb.rope_frequencies(d), nheads=H)
    assert not y[:, 0].any()


@pytest.mark.gpu
def test_many_tokens_sum_the_weights_gradient():
    """More rows than the pullback's blocks take at once, and the same bits each time."""
    d, H, Hk, L, B = 64, 3, 1, 5003, 3
    gen = np.random.default_rng(7)
    q, k, dyq, dyk = (_array(gen, (h * d, L, B), F16) for h in (H, Hk, H, Hk))
    gq, gk = 1 + 0.2 * _array(gen, (d,), F32), 1 + 0.2 * _array(gen, (d,), F32)
    f = nb.rope_frequencies(32)
    _check(q, k, gq, gk, f, H, dyq, dyk)
    a, b = (nb.qk_norm_rope_pullback(q, k, gq, gk, f, nheads=H)[2](dyq, dyk) for _ in range(2))
    assert all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.gpu
def test_empty_batches():
    g, f = torch.ones(16, device=DEV), nb.rope_frequencies(16)
    for L, B in ((0, 2), (3, 0)):
        q, k = nb.jl_empty((32, L, B), F32, DEV), nb.jl_empty((16, L, B), F32, DEV)
        y, yk, back = nb.qk_norm_rope_pullback(q, k, g, g, f, nheads=2)
        assert tuple(y.shape) == (32, L, B) and tuple(yk.shape) == (16, L, B)
        dq, dk, dgq, dgk = back(y, yk)
        assert tuple(dq.shape) == (32, L, B) and not dgq.any() and not dgk.any()


@pytest.mark.gpu
def test_captured_calls_follow_their_positions():
    d, H, L, B = 64, 2, 3, 2
    gen = np.random.default_rng(8)
    q, dy = _array(gen, (H * d, L, B), BF16), _array(gen, (H * d, L, B), BF16)
    g, f = torch.ones(d, device=DEV, dtype=BF16), nb.rope_frequencies(d)
    start = torch.zeros(B, dtype=torch.int32, device=DEV)

    def call():
        y, yk, back = nb.qk_norm_rope_pullback(q, q, g, g, f, nheads=H, start=start)
        return (y, yk, *back(dy, dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = call()
        graphs.append((gr, out))
    for s in ((3, 900), (10, 0)):
        start.copy_(torch.tensor(s, dtype=torch.int32))
        want = call()
        for gr, out in graphs:
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_refusals():
    d, H, L, B = 16, 2, 3, 2
    q, k = nb.jl_zeros((H * d, L, B), F32, DEV), nb.jl_zeros((d, L, B), F32, DEV)
    g, f = torch.ones(d, device=DEV), nb.rope_frequencies(d)
    ok = dict(nheads=H)
    for bad, err in [
        (dict(q=q.cpu()), TypeError), (dict(q=q.double()), TypeError), (dict(k=k.half()), TypeError),
        (dict(q=q[:, :, 0]), TypeError), (dict(k=nb.jl_zeros((d, L + 1, B), F32, DEV)), nb.ArgumentError),
        (dict(k=nb.jl_zeros((d + 1, L, B), F32, DEV)), nb.ArgumentError), (dict(nheads=3), nb.ArgumentError),
        (dict(nheads=0), nb.ArgumentError), (dict(gq=g.half()), TypeError), (dict(gk=g.half()), TypeError),
        (dict(gq=g[:8]), nb.ArgumentError), (dict(freqs=f.float()), TypeError), (dict(freqs=nb.rope_frequencies(18)), nb.ArgumentError),
        (dict(start=torch.zeros(B, device=DEV)), TypeError), (dict(start=torch.zeros(3, dtype=torch.int32, device=DEV)), nb.ArgumentError),
        (dict(positions=torch.zeros((B, L), dtype=torch.int32, device=DEV)), nb.ArgumentError),
        (dict(eps=-1.0), nb.ArgumentError), (dict(eps=float("nan")), nb.ArgumentError),
        (dict(q=q.transpose(0, 1).contiguous().transpose(0, 1)), TypeError),                # features not adjacent
        (dict(q=nb.jl_zeros((H * d, L, 1), F32, DEV).expand(-1, -1, B)), TypeError),
    ]:
        args = dict(q=q, k=k, gq=g, gk=g, freqs=f, **ok) | bad
        a = [args.pop(n) for n in ("q", "k", "gq", "gk", "freqs")]
        with pytest.raises(err):
            nb.qk_norm_rope(*a, **args)
    with pytest.raises(nb._lib.NNlibB200Error):
        w = nb.jl_zeros((258, L, B), F32, DEV)
        nb.qk_norm_rope(w, w, torch.ones(258, device=DEV), torch.ones(258, device=DEV), f, nheads=1)
    _, _, back = nb.qk_norm_rope_pullback(q, k, g, g, f, nheads=H)
    with pytest.raises(nb.ArgumentError):
        back(q[:, :2], k)
    with pytest.raises(TypeError):
        back(q.half(), k)


def test_the_oracles_pullback_agrees_with_differences():
    gen = np.random.default_rng(9)
    d, L, B = 10, 3, 2
    for inter, rot in ((False, 10), (True, 6)):
        x, dy, v = (gen.standard_normal((2 * d, L, B)) for _ in range(3))
        g, vg = gen.standard_normal(d), gen.standard_normal(d)
        f, pos = gen.random(rot // 2), gen.integers(0, 50, (L, B)).astype(float)
        dx, dg = R.pullback(x, g, pos, f, 1e-3, inter, dy)
        h = 1e-5
        num = ((R.norm_rope(x + h * v, g + h * vg, pos, f, 1e-3, inter) - R.norm_rope(x - h * v, g - h * vg, pos, f, 1e-3, inter)) * dy).sum() / (2 * h)
        np.testing.assert_allclose(num, (dx * v).sum() + (dg * vg).sum(), rtol=1e-7)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", [
    # d, rotated, neighbours, query heads, key heads, L, B
    (128, 128, False, 1, 2, 9, 2),        # fewer heads than a warp has groups
    (128, 128, True, 6, 3, 5, 1),         # heads that its groups do not divide
    (80, 80, False, 8, 7, 700, 6),        # six groups, tokens enough that a warp takes all of a token's heads
    (34, 34, False, 3, 2, 6, 2),          # single pairs
    (64, 64, False, 12, 1, 1, 1),         # one token, its heads cut up
])
def test_without_eps(dtype, case):
    """eps = 0: r = 1 / sqrt(mean x^2) of every row that is not all zero, and no trace of rows that a warp does not have."""
    d, rot, inter, H, Hk, L, B = case
    gen = np.random.default_rng(33)
    q, k, dyq, dyk = (_array(gen, (h * d, L, B), dtype) for h in (H, Hk, H, Hk))
    gq, gk = (1 + 0.2 * _array(gen, (d,), F32)).to(dtype), (1 + 0.2 * _array(gen, (d,), F32)).to(dtype)
    _check(q, k, gq, gk, nb.rope_frequencies(rot), H, dyq, dyk, inter, eps=0.0, start=3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d,rot,inter", [(64, 32, False), (64, 32, True), (64, 20, True), (34, 10, False), (254, 20, True), (48, 0, False)])
def test_features_that_are_not_turned_meet_no_others(dtype, d, rot, inter):
    """An infinity in a feature behind the rotated ones: r is 0 and so is every other feature of y; in the cotangent it
    reaches dx of its row, through the mean, and the gradient of its own weight only."""
    H, L, B = 3, 5, 2
    gen = np.random.default_rng(38)
    g, f = (1 + 0.2 * _array(gen, (d,), F32)).to(dtype), nb.rope_frequencies(rot)
    for at in {rot, (rot + d) // 2, d - 1}:
        q, dy = _array(gen, (H * d, L, B), dtype), _array(gen, (H * d, L, B), dtype)
        want = nb.qk_norm_rope(q, q, g, g, f, nheads=H, interleaved=inter, start=4)[0]
        bad = q.clone()
        bad[d + at, 2, 1] = float("inf")
        y, _, back = nb.qk_norm_rope_pullback(bad, bad, g, g, f, nheads=H, interleaved=inter, start=4)
        row = y[d:2 * d, 2, 1]
        assert torch.isnan(row[at]) and not torch.cat((row[:at], row[at + 1:])).float().abs().any()
        same = torch.ones_like(y, dtype=torch.bool)
        same[d:2 * d, 2, 1] = False
        assert torch.equal(y[same], want[same])
        loud = dy.clone()
        loud[d + at, 2, 1] = float("inf")
        dgq = nb.qk_norm_rope_pullback(q, q, g, g, f, nheads=H, interleaved=inter, start=4)[2](loud, dy)[2]
        hit = ~torch.isfinite(dgq.float())
        assert hit[at] and hit.sum().item() == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("inter", [False, True])
def test_float32_gradients_of_the_weights_of_16_bit_arrays(dtype, inter):
    """One row, so that nothing averages out: dg = u x r with u = a cos + b sin of two elements of the cotangent.  The turn is a
    Float32 below 1/2 (2^-26 of a turn, 2^-23.35 as an angle), sine and cosine are within one unit, 2^-24 below 1, and one product
    is rounded: u is off by (|a| + |b|) (2^-23.35 + 2^-24 + 2^-24) < 2^-22.1 (|a| + |b|).  The sum u, r (two units, and the sum
    of squares) and the products by it: 2^-24 + 2^-22 + 2^-23 + 2 * 2^-24 < 2^-21 of the result."""
    d = 128
    gen = np.random.default_rng(41)
    f, g = nb.rope_frequencies(d), 1 + 0.2 * _array(gen, (d,), F32)
    g64, f64 = _f64(g), f.cpu().numpy()
    for at in list(range(40)) + [1000, 77777]:
        x, dy = _array(gen, (d, 1, 1), dtype), _array(gen, (d, 1, 1), dtype)
        got = nb.qk_norm_rope_pullback(x, x, g, g, f, nheads=1, interleaved=inter, start=at)[2](dy, dy)
        pos = np.full((1, 1), float(at))
        _, dg = R.pullback(_f64(x), g64, pos, f64, 1e-6, inter, _f64(dy))
        a = np.abs(_f64(dy)[:, 0, 0])
        both = a + (a.reshape(-1, 2)[:, ::-1].reshape(-1) if inter else np.roll(a, d // 2))
        xr = np.abs(_f64(x)[:, 0, 0]) / np.sqrt((_f64(x) ** 2).mean() + 1e-6)
        for s in got[2:]:
            over = np.abs(_f64(s) - dg) - 2.0 ** -22.1 * both * xr - 2.0 ** -21 * np.abs(dg)
            assert over.max() <= 0, (at, over.max())
