"""The 8-bit key / value cache and attention over it against the oracle.

Scales and codes are Float32 arithmetic that the definition spells out, so they are compared for equality.  Attention:
weights are rounded to Float16 (11 significant bits: half a step is 2^-11 of the value; two terms, 2^-22, for Float32
arrays), which changes x by at most that
times sum p |v| (``size`` below) in the numerator; logits are Float32 sums of at most 256 products of codes and of what 2^13
times a query's element is (Float32: its first 22 bits), off by at most 2^-18 of sum |q||k| scale, which changes a weight
relatively by that, and x by twice that times ``size``; exponentials, page scales and Float32 sums: 2^-19 of ``size``.
Products of a weight and a value scale are multiples of 2^-34 of the largest one (2^-38 where queries are few), so each is off
by 2^-35 of that at least, and x by 2^-35 times ``grid``.  With N(0, 1) inputs sum |q||k| scale <= 0.7 d / sqrt(d) <= 12.  So |x - x64| <= (W + 2 * 12 * 2^-18 + 2^-19) size + 2^-35 grid +
half a step of the result: 2^-11 + 2^-13 for 16-bit arrays, 2^-13 for Float32 ones (which stay far below it)."""
import ctypes as C

import numpy as np
import pytest
import torch

import nnlib_jl_b200 as nb
from oracle import cache_oracle as O

DEV = torch.device("cuda:0")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
NAN, INF = float("nan"), float("inf")
gpu = pytest.mark.gpu


def _i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device=DEV)


def _array(gen, shape, dtype, scale=1.0):
    return (scale * nb.jl_from_numpy(gen.standard_normal(shape).astype(np.float32), device=DEV)).to(dtype)


def _np(t):
    return nb.jl_to_numpy(t.float())


class Pair:
    """A cache on the device and its restatement."""

    def __init__(self, dim, capacity, batch, nheads, page, code, gen, paged):
        self.code, self.batch = code, batch
        rows = -(-capacity // page)
        self.table = None
        if paged:
            order = gen.permutation(batch * rows + 3)[:batch * rows].reshape(rows, batch)
            self.table = np.asarray(order, np.int32)
        self.dev = nb.QuantizedCache(dim, page * (rows * batch + 3) if paged else capacity, 1 if paged else batch,
                                     nheads=nheads, page=page, eltype=CODE[code], device=DEV)
        P = self.dev.pages
        self.codes = [np.zeros((dim, page, P), np.float32) for _ in range(2)]
        self.scale = [np.zeros((nheads, P), np.float32) for _ in range(2)]

    @property
    def t(self):
        return None if self.table is None else nb.jl_from_numpy(self.table, device=DEV)

    def write(self, k, v, start, count=None):
        s = np.full(self.batch, start) if np.isscalar(start) else np.asarray(start)
        nb.cache_write_(self.dev, k, v, start=start if np.isscalar(start) else _i32(start), table=self.t,
                        count=None if count is None else _i32(count))
        for n, x in enumerate((k, v)):
            O.write(self.codes[n], self.scale[n], _np(x), s, self.code, count=count, table=self.table)

    def same(self):
        d = self.dev
        for got, want in zip((d.k, d.v, d.k_scale, d.v_scale), self.codes + self.scale):
            np.testing.assert_array_equal(_np(got), want)

    def attend(self, q, lens, nheads, start=None, causal=True, scale=None):
        L = [int(n) for n in lens]
        x, lse = nb.cached_attention(q, self.dev, _i32(lens), nheads=nheads, table=self.t, causal=causal, scale=scale,
                                     start=None if start is None else _i32(start), return_lse=True)
        want = O.attention(_np(q), *self.codes, *self.scale, L, nheads, start=start, causal=causal, scale=scale, table=self.table)
        check_attention(x, lse, want, q.dtype)
        return x, lse


def check_attention(x, lse, want, dtype):
    x64, lse64, size, grid = want
    got, gl = nb.jl_to_numpy(x.double()), nb.jl_to_numpy(lse.double())
    lim = (2.0 ** -13 if dtype == F32 else 2.0 ** -11 + 2.0 ** -13) * size + 2.0 ** -35 * grid + torch.finfo(dtype).eps / 2 * np.abs(x64) * 1.001
    lim += 2.0 ** -25 if dtype == F16 else 0
    np.testing.assert_array_equal(np.isnan(got), np.isnan(x64))
    ok = ~np.isnan(x64)
    assert (np.abs(got - x64)[ok] <= lim[ok]).all(), float((np.abs(got - x64) - lim)[ok].max())
    np.testing.assert_array_equal(np.isnan(gl), np.isnan(lse64))
    np.testing.assert_array_equal(np.isneginf(gl), np.isneginf(lse64))
    fin = np.isfinite(lse64)
    np.testing.assert_allclose(gl[fin], lse64[fin], atol=2 * 12 * 2.0 ** -18, rtol=2.0 ** -20)


# ------------------------------------------------------------------------------------------------ writing and reading
@gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim,nheads,page,paged", [(32, 2, 16, False), (80, 1, 64, True), (384, 3, 32, True), (512, 2, 256, False),
                                                   (112, 7, 16, True), (256, 2, 128, True)])
def test_writes_match_the_definition(code, dtype, dim, nheads, page, paged):
    """A prompt, single tokens, a run across pages, and one that goes back; every code and scale of the pool."""
    gen = np.random.default_rng(1)
    B, cap = 3, 2 * page + 40
    c = Pair(dim, cap, B, nheads, page, code, gen, paged)
    start = np.array([0, 0, 0])
    for L, scale in ((page + 3, 1.0), (1, 3.0), (1, 0.1), (page // 2, 5.0), (2, 20.0)):
        c.write(_array(gen, (dim, L, B), dtype, scale), _array(gen, (dim, L, B), dtype, 0.3 * scale), start)
        c.same()
        start = start + L + np.array([0, 1, 0])
    c.write(_array(gen, (dim, 7, B), dtype, 50.0), _array(gen, (dim, 7, B), dtype), np.array([3, page, page + 5]))
    c.same()
    for s, n in ((0, cap), (np.array([1, 5, 2]), 9)):
        at = np.full(B, s) if np.isscalar(s) else s
        k, v = nb.cache_read(c.dev, n, start=_i32(at), table=c.t, dtype=dtype)
        for got, codes, scale in zip((k, v), c.codes, c.scale):
            want = torch.from_numpy(O.read(codes, scale, n, at, B, table=c.table)).to(dtype).float().numpy()
            np.testing.assert_array_equal(_np(got), want)


@gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("paged", [False, True])
def test_ragged_writes_edges_and_bad_pages(code, paged):
    """Counts of zero and beyond the length, starts behind the capacity and below zero, pages that the pool does not have."""
    gen = np.random.default_rng(2)
    B, dim, T = 6, 64, 16
    c = Pair(dim, 48, B, 2, T, code, gen, paged)
    if paged:
        c.table[1, 1], c.table[0, 2], c.table[2, 0] = -1, 10 ** 6, c.dev.pages
    k, v = _array(gen, (dim, 40, B), BF16), _array(gen, (dim, 40, B), BF16)
    c.write(k, v, np.array([0, 5, 9, 30, 48, -2]), count=np.array([40, 33, 40, 99, 5, 20]))
    c.same()
    c.write(k[:, :1], v[:, :1], np.array([40, 0, 47, 15, 16, 2 ** 31 - 1]), count=np.array([1, 0, 1, 1, -3, 1]))
    c.same()
    at, lens = np.array([0, -4, 30, 8, 0, 40]), np.array([48, 30, 40, 0, 100, 45])
    got = nb.cache_read(c.dev, 30, start=_i32(at), lens=_i32(lens), table=c.t, dtype=F32)
    for g, codes, scale in zip(got, c.codes, c.scale):
        np.testing.assert_array_equal(_np(g), O.read(codes, scale, 30, at, B, lens=lens, table=c.table))


@gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_values_that_are_not_finite_zero_or_tiny(code):
    gen = np.random.default_rng(3)
    dim, T = 32, 16
    c = Pair(dim, 64, 1, 2, T, code, gen, False)
    k = _array(gen, (dim, 20, 1), F32)
    k[3, 2], k[20, 17] = NAN, -INF                       # head 0 of page 0, head 1 of page 1
    v = _array(gen, (dim, 20, 1), F32, 1e-41)            # the scales would be below 2^-126
    v[:16, 16:] = 0
    c.write(k, v, 0)
    c.same()
    more = _array(gen, (dim, 3, 1), F32)
    c.write(more, more, 20)                              # the poisoned block stays, the zero one takes its first scale
    c.same()
    assert np.isnan(c.scale[0][0, 0]) and np.isnan(c.scale[0][1, 1]) and c.scale[0][1, 0] > 0 and c.scale[1][0, 0] == 0
    c.write(more, more, 0)                               # begun anew
    c.same()
    assert np.isfinite(c.scale[0][0, 0])
    big = _array(gen, (dim, 2, 1), F32, 1e38)
    c.write(big, big, 32)
    c.same()


@gpu
def test_views_and_other_pages_are_left_alone():
    """k and v as slices of a projection, at any alignment; what the call does not write keeps its bits."""
    gen = np.random.default_rng(4)
    dim, T, B = 48, 16, 2
    for dtype, shift in ((BF16, 0), (BF16, 1), (F32, 1), (F16, 3)):
        c = Pair(dim, 64, B, 3, T, "int8", gen, True)
        junk = gen.integers(-127, 128, c.codes[0].shape).astype(np.float32)
        for n, t in enumerate((c.dev.k, c.dev.v)):
            t.copy_(nb.jl_from_numpy(junk, device=DEV))
            c.codes[n][:] = junk
        packed = _array(gen, (3 * dim + 5, 21, B), dtype)
        c.write(packed[dim + shift:2 * dim + shift], packed[2 * dim + shift:3 * dim + shift], np.array([7, 20]))
        c.same()


# ------------------------------------------------------------------------------------------------ attention
def _filled(gen, dim, cap, B, H, page, code, paged, dtype=BF16):
    c = Pair(dim, cap, B, H, page, code, gen, paged)
    c.write(_array(gen, (dim, cap, B), dtype), _array(gen, (dim, cap, B), dtype, 0.5), 0)
    return c


@gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d,Hq,H,L,cap,page,paged", [
    (64, 12, 12, 1, 500, 16, False),
    (128, 8, 2, 1, 300, 64, True),
    (128, 4, 4, 3, 700, 128, True),
    (16, 2, 1, 1, 33, 16, False),
    (80, 6, 2, 5, 130, 32, True),          # 15 rows of a tile, features between the padded sizes
    (112, 5, 1, 4, 100, 16, True),         # 20 rows: more than one tile
    (48, 16, 2, 33, 65, 32, False),        # 264 rows
    (256, 2, 2, 2, 90, 64, True),
    (160, 9, 3, 7, 50, 16, True),
    (96, 1, 1, 64, 64, 64, False),         # a whole prompt over itself
    (128, 32, 8, 130, 400, 64, True),      # 520 rows
])
def test_attention_matches_the_oracle(code, dtype, d, Hq, H, L, cap, page, paged):
    gen = np.random.default_rng(5)
    B = 2
    c = _filled(gen, d * H, cap, B, H, page, code, paged)
    q = _array(gen, (d * Hq, L, B), dtype)
    c.attend(q, [cap, max(L, cap // 2 + 1)], Hq)
    c.attend(q, [cap - 1, 1], Hq, causal=False, scale=0.3)


def _path(c, q, nheads):
    """Which kernels a call with lengths on the device takes."""
    k = c.dev._call(q.shape[2], c.t)
    p = nb._lib.CacheAttnParams(dtype=nb.attention._DTYPES[q.dtype], causal=1, Hq=nheads, L=q.shape[1], q=0x1000, x=0x1000, lens=0x1000)
    return nb._lib.load().nnlib_b200_cache_attn_path(C.byref(k), C.byref(p))


@gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,Hq,H,L,cap,page,paged", [
    (16, 64, 64, 60, 380, 16, True),       # heads enough that few queries and keys make a large call
    (64, 64, 64, 33, 530, 64, False),
    (64, 96, 48, 33, 400, 32, True),
    (80, 64, 64, 30, 490, 16, False),
    (112, 64, 32, 300, 300, 128, True),    # 600 rows: three blocks, the last one's second tile empty
    (128, 64, 64, 129, 1100, 64, True),    # keys cut into parts
    (128, 48, 16, 90, 520, 32, True),
])
def test_attention_on_the_tensor_cores_matches_the_oracle(code, dtype, d, Hq, H, L, cap, page, paged):
    gen = np.random.default_rng(15)
    B = 2 if L < 200 else 1
    c = _filled(gen, d * H, cap, B, H, page, code, paged)
    q = _array(gen, (d * Hq, L, B), dtype)
    assert _path(c, q, Hq) == nb._lib.PATH_UMMA
    c.attend(q, [cap, max(L, cap // 2 + 1)][:B], Hq)
    c.attend(q, [cap - 1, 1][:B], Hq, causal=False, scale=0.3)
    nb.device_health()


@gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("page", [16, 64])
def test_tensor_cores_with_lengths_of_every_kind(code, page):
    gen = np.random.default_rng(16)
    d, H, L, cap, B = 16, 64, 45, 200, 7
    c = _filled(gen, d * H, cap, B, H, page, code, True)
    q = _array(gen, (d * H, L, B), BF16)
    assert _path(c, q, H) == nb._lib.PATH_UMMA
    lens = [0, 1, 31, 33, 10 ** 9, -5, 150]
    c.attend(q, lens, H)
    c.attend(q, lens, H, causal=False)
    x, lse = c.attend(q, lens, H, start=[0, -2, 40, 2, 190, 0, -L - 3])
    assert torch.isnan(x[:, :, 6].float()).all() and torch.isneginf(lse[:, :, 6]).all()


@gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_tensor_cores_and_what_a_query_does_not_see(code):
    """Poisoned and missing pages, E4M3's NaN behind the last token, as in the test for few queries below."""
    gen = np.random.default_rng(17)
    d, H, L, T = 32, 64, 50, 16
    c = _filled(gen, d * H, 320, 3, H, T, code, True)
    c.dev.v_scale[:, c.table[18, 0]], c.scale[1][:, c.table[18, 0]] = NAN, NAN
    c.dev.k_scale[:, c.table[17, 1]], c.scale[0][:, c.table[17, 1]] = NAN, NAN
    c.table[19, 2] = -1
    if code == "e4m3":
        for n, t in enumerate((c.dev.k, c.dev.v)):
            t.view(torch.uint8)[:, 9:, c.table[18, 1]] = 0x7f
            c.codes[n][:, 9:, c.table[18, 1]] = NAN
    q = _array(gen, (d * H, L, 3), F16)
    assert _path(c, q, H) == nb._lib.PATH_UMMA
    x, _ = c.attend(q, [304, 297, 319], H)               # queries 254 .., 247 .. and 269 ..
    assert torch.isfinite(x[:, 0].float()).all() and torch.isnan(x[:, -1, 0].float()).all()
    c.attend(q, [288, 16 * 17, 304], H)


@gpu
def test_tensor_cores_captured_with_lengths_that_change():
    gen = np.random.default_rng(18)
    d, H, L, B = 64, 64, 40, 2
    c = _filled(gen, d * H, 700, B, H, 64, "int8", True)
    q, lens, t = _array(gen, (d * H, L, B), BF16), _i32([60, 700]), c.t
    assert _path(c, q, H) == nb._lib.PATH_UMMA
    want = nb.cached_attention(q, c.dev, lens, nheads=H, table=t)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x = nb.cached_attention(q, c.dev, lens, nheads=H, table=t)
    for n in ([60, 700], [40, 333], [699, 41]):
        lens.copy_(_i32(n))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, nb.cached_attention(q, c.dev, lens, nheads=H, table=t))
    lens.copy_(_i32([60, 700]))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(x, want)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("L", [1, 3, 20, 150])
def test_lengths_of_every_kind(code, dtype, L):
    """No tokens, one, a length that ends inside a page, beyond the capacity; starts that leave queries without a token."""
    gen = np.random.default_rng(6)
    d, H, Hq, cap = 64, 2, 4, 200
    B = 7
    c = _filled(gen, d * H, cap, B, H, 32, code, True)
    q = _array(gen, (d * Hq, L, B), dtype)
    lens = [0, 1, 31, 33, 10 ** 9, -5, 150]
    c.attend(q, lens, Hq)
    c.attend(q, lens, Hq, causal=False)
    x, lse = c.attend(q, lens, Hq, start=[0, -2, 40, 2, 190, 0, -L - 3])
    assert torch.isnan(x[:, :, 6].float()).all() and torch.isneginf(lse[:, :, 6]).all()


@gpu
@pytest.mark.parametrize("L", [2, 40, 140])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_a_query_does_not_see_does_not_reach_it(code, dtype, L):
    """NaN codes and NaN scales behind the last token, poisoned and missing pages that only later queries see."""
    gen = np.random.default_rng(7)
    d, H, Hq, T = 128, 1, 3, 16
    c = _filled(gen, d * H, 320, 3, H, T, code, True)
    c.dev.v_scale[:, c.table[18, 0]], c.scale[1][:, c.table[18, 0]] = NAN, NAN       # tokens 288 .. 303
    c.dev.k_scale[:, c.table[17, 1]], c.scale[0][:, c.table[17, 1]] = NAN, NAN
    c.table[19, 2] = -1
    if code == "e4m3":      # whatever a slot held before: E4M3's NaN behind the last token of sequence 1
        for n, t in enumerate((c.dev.k, c.dev.v)):
            t.view(torch.uint8)[:, 9:, c.table[18, 1]] = 0x7f
            c.codes[n][:, 9:, c.table[18, 1]] = NAN
    q = _array(gen, (d * Hq, L, 3), dtype)
    lens = [288 + min(L // 2, 16), 297, 304 + min(L // 2, 15)]
    x, _ = c.attend(q, lens, Hq)
    assert torch.isfinite(x[:, 0, 0].float()).all() and torch.isnan(x[:, -1, 0].float()).all()
    c.attend(q, [288, 16 * 17, 304], Hq)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_scales_far_apart_and_large_logits(dtype):
    """Pages whose values differ by 2^60 and more, logits of several hundred, and a first page that later ones dwarf."""
    gen = np.random.default_rng(8)
    d, T = 64, 16
    c = _filled(gen, d, 160, 1, 1, T, "int8", False, F32)
    f = np.float32([1, 2.0 ** -60, 2.0 ** 20, 1, 2.0 ** -20, 0, 2.0 ** -90, 1, 4, 2.0 ** 10]) * (2.0 ** -10 if dtype == F16 else 1)
    c.scale[1] *= f
    c.dev.v_scale.copy_(nb.jl_from_numpy(c.scale[1], device=DEV))
    for L, size in ((1, 1.0), (5, 1.0), (64, 1.0)):
        q = _array(gen, (d, L, 1), dtype, size)
        for n in (16, 32, 33, 48, 100, 160):
            c.attend(q, [max(n, L)], 1)
    # large logits: a weight of one and the rest nothing, exactly representable so that the logits are
    c = _filled(gen, d, 160, 1, 1, T, "int8", False, F32)
    q = _array(gen, (d, 2, 1), dtype, 40.0)
    x = nb.cached_attention(q, c.dev, 160, nheads=1)
    want = O.attention(_np(q), *c.codes, *c.scale, [160], 1)
    # logits of size 300 are off by 300 * 2^-18 at most, weights by twice that
    over = np.abs(nb.jl_to_numpy(x.double()) - want[0]) - (2.0 ** -8) * want[2] - 2.0 ** -35 * want[3]
    assert over.max() <= 0, over.max()


@gpu
def test_queries_out_of_the_ordinary():
    gen = np.random.default_rng(9)
    d, H = 64, 2
    c = _filled(gen, d * H, 100, 1, H, 32, "int8", False)
    q = _array(gen, (d * H, 4, 1), F32)
    q[:, 1] *= 1e30
    q[:64, 0] = 0
    q[64:, 2] *= 1e-40
    q[3, 3], q[70, 3] = NAN, INF
    x = nb.cached_attention(q, c.dev, 100, nheads=H, scale=1e-30)
    assert torch.isfinite(x[:, :3]).all() and torch.isnan(x[:, 3]).all()
    want = O.attention(_np(q)[:, :3], *c.codes, *c.scale, [99], H, start=[96], scale=1e-30)
    got = nb.jl_to_numpy(x.double())[:, [0, 2]]
    over = np.abs(got - want[0][:, [0, 2]]) - 2.0 ** -13 * want[2][:, [0, 2]] - 2.0 ** -35 * want[3][:, [0, 2]]
    assert over.max() <= 0, over.max()


@gpu
def test_strided_queries_and_other_layouts():
    gen = np.random.default_rng(10)
    d, H, Hq, B = 32, 2, 4, 2
    c = _filled(gen, d * H, 90, B, H, 16, "e4m3", True)
    for dtype in (BF16, F32):
        for shift in (0, 1, 2):
            packed = _array(gen, (d * Hq + 7, 6, B), dtype)
            c.attend(packed[shift:shift + d * Hq], [90, 40], Hq)


@gpu
def test_a_pool_past_32_bits():
    """Codes and scales of pages whose offset passes 2^31, and 2^32, bytes."""
    gen = np.random.default_rng(11)
    dim, H, T, P = 1024, 8, 64, 70000                                # 4.6 GB of codes each
    cache = nb.QuantizedCache(dim, T * P, nheads=H, page=T, device=DEV)
    pages = np.array([[69999, 3], [40000, 65536], [32768, 69998]], np.int32)
    t = nb.jl_from_numpy(pages, device=DEV)
    k, v = _array(gen, (dim, 150, 2), BF16), _array(gen, (dim, 150, 2), BF16)
    nb.cache_write_(cache, k, v, table=t)
    small = Pair(dim, 192, 2, H, T, "int8", gen, False)
    small.write(k, v, 0)
    got, want = nb.cache_read(cache, 150, table=t, dtype=F32), nb.cache_read(small.dev, 150, dtype=F32)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for L in (1, 70):
        q = _array(gen, (dim, L, 2), BF16)
        assert torch.equal(nb.cached_attention(q, cache, 150, nheads=H, table=t), nb.cached_attention(q, small.dev, 150, nheads=H))


@gpu
def test_a_long_history():
    """Many shares of one unit, against the framework's own attention on the tokens read back."""
    gen = torch.Generator(device="cuda").manual_seed(12)
    d, H, n = 128, 2, 40001
    cache = nb.QuantizedCache(d * H, n, nheads=H, page=64, device=DEV)
    k, v = nb.jl_empty((d * H, n, 1), F16, DEV).normal_(generator=gen), nb.jl_empty((d * H, n, 1), F16, DEV).normal_(generator=gen)
    nb.cache_write_(cache, k, v)
    kr, vr = nb.cache_read(cache, n, dtype=F32)
    for L in (1, 4, 70):
        q = nb.jl_empty((d * H, L, 1), F16, DEV).normal_(generator=gen)
        x = nb.cached_attention(q, cache, n, nheads=H)
        want, _ = nb.dot_product_attention(q.float(), kr, vr, mask=nb.CausalMask(n - L), nheads=H)
        # sum p |v| is at most 1 here, and rounding errors of 40000 weights partly cancel
        assert (x.float() - want).abs().max().item() <= 2.0 ** -11 + 2.0 ** -13


@gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_float32_sums_of_a_long_history_are_rounded(code):
    """Positive values behind 131072 keys: a warp adds up to N = 131072 / 64 steps to a sum, and each addition that rounds is off
    by at most 2^-24 of it, to either side: 5 sqrt(N / 3) 2^-24 at five standard deviations, once for x and once for the sum of
    the weights; 8 2^-24 for the weights' two terms, a step's products and what the read values are rounded by.  Additions
    that cut off would shrink every element alike, by up to N 2^-23.  The logits' own error, 2 * 2^-18 sum |q||k| scale at
    most, moves elements to both sides; q is small, so that this stays below 8 2^-24 too."""
    d, Hq, L, n = 32, 8, 1024, 131072
    gen = np.random.default_rng(77)
    c = nb.QuantizedCache(d, n, 1, nheads=1, page=64, eltype=CODE[code], device=DEV)
    k, v = _array(gen, (d, n, 1), F32), _array(gen, (d, n, 1), F32)
    nb.cache_write_(c, k, v.abs() + 0.5)
    q = _array(gen, (d * Hq, L, 1), F32, 2.0 ** -7)
    x = nb.cached_attention(q, c, n, nheads=Hq, causal=False)
    kr, vr = (t[:, :, 0].double() for t in nb.cache_read(c, n, dtype=F32))
    at = torch.arange(0, L, 33, device=DEV)
    rows = q[:, at, 0].double().reshape(Hq, d, -1)
    want = torch.stack([torch.softmax(r.T @ kr / d ** 0.5, 1) @ vr.T for r in rows])            # (Hq, rows, d)
    got = x[:, at, 0].double().reshape(Hq, d, -1).transpose(1, 2)
    lim = (2 * 5 * (n / 64 / 3) ** 0.5 + 16) * 2.0 ** -24
    off = got / want - 1
    assert off.abs().max().item() <= lim, (off.abs().max().item(), off.mean().item(), lim)


@gpu
@pytest.mark.parametrize("L", [3, 1024])
def test_float16_sums_of_a_very_long_history(L):
    """Positive values behind 524288 keys: sum p |v| is x itself here.  Weights' roundings fall to both sides and cancel
    over so many; 2^-12 for the sums (blocks of 32768 keys, each key's part of a cut-off addition 2^-27), half a step of the result, 2^-11."""
    d, Hq, n = 32, 8, 524288
    gen = torch.Generator(device="cuda").manual_seed(5)
    c = nb.QuantizedCache(d, n, 1, nheads=1, page=64, eltype=torch.int8, device=DEV)
    k, v = (nb.jl_empty((d, n, 1), F16, DEV).normal_(generator=gen) for _ in range(2))
    nb.cache_write_(c, k, v.abs() + 0.5)
    q = nb.jl_empty((d * Hq, L, 1), F16, DEV).normal_(generator=gen) * 2.0 ** -7
    x = nb.cached_attention(q, c, n, nheads=Hq, causal=False)
    kr, vr = (t[:, :, 0].double() for t in nb.cache_read(c, n, dtype=F32))
    at = torch.arange(0, L, 61, device=DEV)
    rows = q[:, at, 0].double().reshape(Hq, d, -1)
    want = torch.stack([torch.softmax(r.T @ kr / d ** 0.5, 1) @ vr.T for r in rows])
    off = x[:, at, 0].double().reshape(Hq, d, -1).transpose(1, 2) / want - 1
    # what is common to all elements is what the sums lose, 32768 2^-27 at most; the results' roundings, 32 different ones
    # where queries are nearly alike, leave 2^-11 / sqrt(3 * 32) at one standard deviation
    far = off.abs().max().item()
    assert far <= 2.0 ** -11 + 2.0 ** -12
    mean = abs(off.mean().item())
    assert mean <= 2.0 ** -12 + 3 * 2.0 ** -11 / 96 ** 0.5


@gpu
def test_capture_replay_streams_and_repeatability():
    gen = np.random.default_rng(13)
    d, H, Hq, B = 64, 2, 8, 3
    c = _filled(gen, d * H, 300, B, H, 32, "int8", True)
    q, k, v = (_array(gen, (d * h, 1, B), BF16) for h in (Hq, H, H))
    start, lens, t = _i32([5, 100, 200]), _i32([6, 101, 201]), c.t

    def step():
        nb.cache_write_(c.dev, k, v, start=start, table=t)
        return nb.cached_attention(q, c.dev, lens, nheads=Hq, table=t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, step())
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x = step()
        graphs.append((g, x))
    for n in (7, 31, 32, 64):
        start.copy_(_i32([n, 100 + n, 200 + n]))
        lens.copy_(start + 1)
        k.copy_(_array(gen, (d * H, 1, B), BF16, 1.0 + n))
        q.copy_(_array(gen, (d * Hq, 1, B), BF16))
        for g, x in graphs:
            x.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(x, step())
    # both graphs' calls at once, on streams of their own (the pages they write are the same, with the same tokens)
    want = step()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (g, x) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for _, x in graphs)


@gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_a_decoder_layers_steps(code):
    """Prompt and generated tokens through norm, rotation, cache and attention, against the framework's own attention over
    what the cache holds."""
    gen = np.random.default_rng(14)
    d, Hq, H, B, prompt = 64, 4, 2, 3, 45
    g = (1 + 0.1 * _array(gen, (d,), F32)).to(BF16)
    f = nb.rope_frequencies(d)
    cache = nb.QuantizedCache(d * H, 96, B, nheads=H, page=16, eltype=CODE[code], device=DEV)
    at = 0
    for L in (prompt, 1, 1, 5, 1):
        packed = _array(gen, ((Hq + 2 * H) * d, L, B), BF16)
        q, k, v = packed[:Hq * d], packed[Hq * d:(Hq + H) * d], packed[(Hq + H) * d:]
        start = _i32([at] * B)
        q, k = nb.qk_norm_rope(q, k, g, g, f, nheads=Hq, start=start)
        nb.cache_write_(cache, k, v, start=start)
        x = nb.cached_attention(q, cache, at + L, nheads=Hq)
        at += L
        kr, vr = nb.cache_read(cache, at, dtype=F32)
        wide = [t.permute(2, 1, 0).reshape(B, at, H, 1, d).expand(-1, -1, -1, Hq // H, -1).reshape(B, at, Hq * d).permute(2, 1, 0)
                for t in (kr, vr)]
        want, _ = nb.dot_product_attention(q.float(), *wide, mask=nb.CausalMask(at - L), nheads=Hq)
        assert torch.allclose(x.float(), want, rtol=2.0 ** -8, atol=(2.0 ** -11 + 2.0 ** -13) * 4)
    # what the layer was given is what it read back, to a code's step
    assert (kr[:, -1].double() - k[:, -1].double()).abs().max().item() <= (4 / 254 + 4 / 256 if code == "int8" else 4 / 16)


@gpu
def test_refusals():
    c = nb.QuantizedCache(64, 64, 2, nheads=2, page=16, device=DEV)
    k = nb.jl_zeros((64, 3, 2), BF16, DEV)
    bad = nb.ArgumentError
    for args, err in [
        (dict(k=k.cpu()), TypeError), (dict(v=k.float()), TypeError), (dict(k=nb.jl_zeros((32, 3, 2), BF16, DEV)), bad),
        (dict(v=nb.jl_zeros((64, 2, 2), BF16, DEV)), bad), (dict(start=_i32([0])), bad), (dict(start=torch.zeros(2, device=DEV)), TypeError),
        (dict(count=_i32([0, 0, 0])), bad), (dict(count=torch.zeros(2, dtype=torch.int64, device=DEV)), TypeError),
        (dict(table=_i32([[0, 1], [2, 3]])), bad),                                       # row-major
        (dict(table=torch.zeros((4, 2), device=DEV)), TypeError), (dict(table=_i32([[0], [1]])), bad),
        (dict(k=k.transpose(0, 1).contiguous().transpose(0, 1)), TypeError),
    ]:
        with pytest.raises(err):
            a = dict(k=k, v=k) | args
            nb.cache_write_(c, a.pop("k"), a.pop("v"), **a)
    for args, err in [(dict(length=-1), bad), (dict(dtype=torch.float64), TypeError), (dict(lens=_i32([1])), bad),
                      (dict(table=_i32([0, 1])), TypeError)]:
        with pytest.raises(err):
            nb.cache_read(c, **(dict(length=4, start=_i32([0, 0])) | args))
    q = nb.jl_zeros((128, 1, 2), BF16, DEV)
    for args, err in [(dict(nheads=3), bad), (dict(nheads=2), bad), (dict(nheads=0), bad), (dict(q=q.double()), TypeError),
                      (dict(q=q[:, 0]), TypeError), (dict(lens=_i32([1])), bad), (dict(lens=torch.zeros(2, device=DEV)), TypeError),
                      (dict(start=_i32([1, 2, 3])), bad), (dict(scale=0.0), bad), (dict(scale=-1.0), bad), (dict(scale=INF), bad),
                      (dict(scale=NAN), bad)]:
        with pytest.raises(err):
            a = dict(q=q, lens=3, nheads=4) | args
            nb.cached_attention(a.pop("q"), c, a.pop("lens"), **a)
    for args, err in [(dict(page=24), bad), (dict(page=8), bad), (dict(page=512), bad), (dict(nheads=3), bad), (dict(eltype=torch.uint8), TypeError)]:
        with pytest.raises(err):
            nb.QuantizedCache(64, 64, **(dict(nheads=2, device=DEV) | args))
    with pytest.raises(nb._lib.NNlibB200Error):                                          # head size 24
        w = nb.QuantizedCache(48, 64, 2, nheads=2, device=DEV)
        nb.cache_write_(w, nb.jl_zeros((48, 1, 2), BF16, DEV), nb.jl_zeros((48, 1, 2), BF16, DEV))
    a = (c.k, c.v, c.k_scale, c.v_scale)
    for n, t in ((1, c.v[:, :, :4]), (2, c.k_scale.half()), (2, c.k_scale[:, :3]), (0, c.k.view(torch.uint8)), (3, c.v_scale.cpu()),
                 (3, c.v_scale.contiguous())):
        with pytest.raises((TypeError, bad)):
            nb.QuantizedCache.from_arrays(*a[:n], t, *a[n + 1:])


@gpu
def test_empty_calls():
    c = nb.QuantizedCache(64, 64, 2, nheads=2, page=16, device=DEV)
    e = nb.jl_empty((64, 0, 2), BF16, DEV)
    nb.cache_write_(c, e, e)
    assert tuple(nb.cached_attention(e, c, 3, nheads=2).shape) == (64, 0, 2)
    none = nb.jl_empty((64, 3, 0), BF16, DEV)
    nb.cache_write_(c, none, none)
    assert tuple(nb.cached_attention(none, c, 3, nheads=2).shape) == (64, 3, 0)
    assert tuple(nb.cache_read(c, 0)[0].shape) == (64, 0, 2)
    nothing = nb.QuantizedCache(64, 0, 2, nheads=2, device=DEV)              # no page at all
    k = nb.jl_zeros((64, 3, 2), BF16, DEV)
    nb.cache_write_(nothing, k, k)
    assert not nb.cache_read(nothing, 2)[0].any()
    assert torch.isnan(nb.cached_attention(k, nothing, 3, nheads=2).float()).all()
    assert torch.isnan(nb.cached_attention(k, nothing, 3, nheads=2, table=nb.jl_zeros((4, 2), torch.int32, DEV)).float()).all()


# ------------------------------------------------------------------------------------------------ found later
@gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [144, 176, 208, 240])
def test_heads_whose_last_features_are_half_of_a_lanes_share(code, dtype, d):
    """Heads of more than 128 features that are no multiple of 32; the last token of the pool's last page, with arrays that
    lie inside larger ones whose bytes behind are no numbers.  (The kernel's loads are checked when it is compiled.)"""
    gen = np.random.default_rng(31)
    H, Hq, B, T, cap = 2, 4, 2, 16, 64
    c = Pair(d * H, cap, B, H, T, code, gen, False)
    wide = [torch.full((c.dev.k.numel() + 4096,), 0x7f, dtype=torch.uint8, device=DEV) for _ in range(2)]
    inner = [nb.jl_reshape(w[:c.dev.k.numel()].view(c.dev.k.dtype), c.dev.k.shape) for w in wide]
    c.dev = nb.QuantizedCache.from_arrays(*inner, c.dev.k_scale, c.dev.v_scale, batch=B)
    c.write(_array(gen, (d * H, cap, B), dtype), _array(gen, (d * H, cap, B), dtype, 0.5), 0)
    c.same()
    for L in (1, 3, 20):
        c.attend(_array(gen, (d * Hq, L, B), dtype), [cap, cap - 7], Hq)
    assert all((w[c.dev.k.numel():] == 0x7f).all() for w in wide)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("what", ["value scale", "key scale", "page"])
def test_a_bad_page_counts_beside_a_dominating_logit(what, dtype):
    """The bad page in one block's share of the keys; in another's, logits some 400 above all in the first, whose weight
    beside them is 0 in Float32.  Few tokens to a share: a step of four warps."""
    gen = np.random.default_rng(32)
    d, T, n = 32, 32, 2560
    c = _filled(gen, d, n, 1, 1, T, "int8", True)
    loud, bad = c.table[60, 0], c.table[0, 0]
    c.scale[0][:, loud] *= 200
    c.dev.k_scale[:, loud] *= 200
    if what == "page":
        c.table[0, 0] = -1
    else:
        side = 1 if what == "value scale" else 0
        (c.dev.k_scale, c.dev.v_scale)[side][:, bad], c.scale[side][:, bad] = NAN, NAN
    for L in (1, 3):
        x, lse = c.attend(_array(gen, (d, L, 1), dtype), [n], 1)
        assert torch.isnan(x.float()).all() and torch.isnan(lse).all()


@gpu
def test_a_call_without_a_table_is_for_the_caches_own_sequences():
    gen = np.random.default_rng(34)
    dim, H, T, B, cap = 64, 2, 16, 4, 48
    c = Pair(dim, cap, B, H, T, "int8", gen, False)
    c.write(_array(gen, (dim, cap, B), BF16), _array(gen, (dim, cap, B), BF16), 0)
    for n in (1, 2, 3, 5, 8):
        k = _array(gen, (dim, 5, n), BF16)
        with pytest.raises(nb.ArgumentError):
            nb.cache_write_(c.dev, k, k)
        with pytest.raises(nb.ArgumentError):
            nb.cached_attention(k, c.dev, 5, nheads=H)
        for how in (dict(start=_i32([0] * n)), dict(lens=_i32([1] * n))):
            with pytest.raises(nb.ArgumentError):
                nb.cache_read(c.dev, 3, **how)
    c.same()
    # one sequence does not reach its neighbour's pages
    one = _array(gen, (dim, 20, 4), BF16)
    c.write(one, one, 40)
    c.same()
    # with a table a call is for as many as that has
    k, t = _array(gen, (dim, 5, 1), BF16), nb.jl_from_numpy(np.array([[7], [0]], np.int32), device=DEV)
    nb.cache_write_(c.dev, k, k, table=t)
    assert torch.equal(nb.cache_read(c.dev, 5, table=t)[0], nb.cache_read(c.dev, 5, start=_i32([0, 0, 16, 0]))[0][:, :, 2:3])
    # a pool without a batch of its own goes by the call's
    pool = nb.QuantizedCache.from_arrays(c.dev.k, c.dev.v, c.dev.k_scale, c.dev.v_scale)
    assert pool.batch is None and nb.QuantizedCache.from_arrays(c.dev.k, c.dev.v, c.dev.k_scale, c.dev.v_scale, batch=B).batch == B
    k = _array(gen, (dim, 5, 2), BF16)
    nb.cache_write_(pool, k, k, start=90)
    at, halves = _i32([90, 90]), nb.jl_from_numpy(np.arange(12, dtype=np.int32).reshape(2, 6).T.copy(), device=DEV)
    assert torch.equal(nb.cache_read(pool, 5, start=at)[0], nb.cache_read(pool, 5, start=at, table=halves)[0])
    assert tuple(nb.cache_read(pool, 4)[0].shape) == (dim, 4, 1)
    held = nb.QuantizedCache.from_arrays(c.dev.k, c.dev.v, c.dev.k_scale, c.dev.v_scale, batch=B)
    with pytest.raises(nb.ArgumentError):
        nb.cache_write_(held, k, k)
    with pytest.raises(nb.ArgumentError):
        nb.QuantizedCache.from_arrays(c.dev.k, c.dev.v, c.dev.k_scale, c.dev.v_scale, batch=-1)


@gpu
def test_a_capacity_below_the_run_of_pages():
    """A sequence's pages begin at (pages / B) * b also where the struct's rows, its capacity, are fewer than pages / B."""
    gen = np.random.default_rng(35)
    d, H, T, B = 32, 2, 16, 3
    c = nb.QuantizedCache(d * H, 64, B, nheads=H, page=T, device=DEV)             # four pages each
    k, q = _array(gen, (d * H, 50, B), BF16), _array(gen, (d * H, 1, B), BF16)
    lib, L = nb._lib.load(), nb._lib
    s = c._call(B, None)
    s.rows = 2
    p = L.CacheTokens(dtype=L.BF16, L=50, k=k.data_ptr(), v=k.data_ptr())
    assert lib.nnlib_b200_cache_write(C.byref(s), C.byref(p), None) == L.OK
    torch.cuda.synchronize()
    back = nb.cache_read(c, 50, dtype=F32)[0]
    assert (back[:, :32] - k[:, :32].float()).abs().max().item() <= 5 / 254 and not back[:, 32:].any()
    got = nb.jl_zeros((d * H, 50, B), F32, DEV)
    p = L.CacheTokens(dtype=L.F32, L=50, k=got.data_ptr(), v=got.data_ptr())
    assert lib.nnlib_b200_cache_read(C.byref(s), C.byref(p), None) == L.OK
    x = nb.jl_zeros((d * H, 1, B), BF16, DEV)
    a = L.CacheAttnParams(dtype=L.BF16, causal=0, Hq=H, L=1, q=q.data_ptr(), x=x.data_ptr(), len0=60)
    assert lib.nnlib_b200_cache_attn_workspace_bytes(C.byref(s), C.byref(a)) == 0
    assert lib.nnlib_b200_cache_attn(C.byref(s), C.byref(a), None, 0, None) == L.OK
    torch.cuda.synchronize()
    assert torch.equal(got, back) and torch.equal(x, nb.cached_attention(q, c, 32, nheads=H, causal=False))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("L", [2, 20, 40])
def test_a_missing_page_and_a_pool_whose_first_page_holds_no_numbers(dtype, L):
    """Queries that do not see the missing page are finite, although page 0, which no sequence has, is all NaN codes."""
    gen = np.random.default_rng(36)
    d, H, Hq, T, B = 64, 1, 2, 16, 2
    c = _filled(gen, d * H, 96, B, H, T, "e4m3", True)
    spare = [p for p in range(c.dev.pages) if p not in c.table][0]
    if (c.table == 0).any():                                     # page 0 gives its place to one that is not used
        for t, host in zip((c.dev.k.view(torch.uint8), c.dev.v.view(torch.uint8)), c.codes):
            t[:, :, spare] = t[:, :, 0]
            host[:, :, spare] = host[:, :, 0]
        for t, host in zip((c.dev.k_scale, c.dev.v_scale), c.scale):
            t[:, spare] = t[:, 0]
            host[:, spare] = host[:, 0]
        c.table[c.table == 0] = spare
    for t, host in zip((c.dev.k, c.dev.v), c.codes):
        t.view(torch.uint8)[:, :, 0] = 0x7f
        host[:, :, 0] = NAN
    c.table[5, 0], c.table[3, 1] = -1, 10 ** 6
    q = _array(gen, (d * Hq, L, B), dtype)
    lens = [80 + min(L // 2, 16), 48 + min(L // 2, 16)]
    x, _ = c.attend(q, lens, Hq)
    assert torch.isfinite(x[:, 0].float()).all() and torch.isnan(x[:, -1].float()).all()


@gpu
@pytest.mark.parametrize("loud", [1, 200])
@pytest.mark.parametrize("dtype,n", [(F16, 300032), (BF16, 600064)])
def test_sums_of_a_very_long_history_that_one_block_walks_over(dtype, n, loud):
    """Rows enough that no block's keys are cut into parts; positive values, so that additions that cut off shrink every
    element alike, by 2^-27 of it for each key that the products sum up by themselves: 32768 (Float16), 262144 (BFloat16).
    ``loud``: the last third's logits are that much larger, so that a maximum rises behind sums that have been put aside;
    there sum |q||k| scale <= 9 (0.64 * 200 * 2^-7 * 32 / sqrt(32), half as much again), which moves weights by 2 * 9 * 2^-18 < 2^-13.
    The results' roundings leave half a step / sqrt(3 * 32) in the mean, as in the test above."""
    d, Hq, L = 32, 8, 2400
    gen = torch.Generator(device="cuda").manual_seed(6)
    c = nb.QuantizedCache(d, n, 1, nheads=1, page=64, eltype=torch.int8, device=DEV)
    k, v = (nb.jl_empty((d, n, 1), F16, DEV).normal_(generator=gen) for _ in range(2))
    nb.cache_write_(c, k, v.abs() + 0.5)
    c.k_scale[:, n // 96:] *= loud
    q = (nb.jl_empty((d * Hq, L, 1), F32, DEV).normal_(generator=gen) * 2.0 ** -7).to(dtype)
    x = nb.cached_attention(q, c, n, nheads=Hq, causal=False)
    nb.device_health()
    kr, vr = (t[:, :, 0].double() for t in nb.cache_read(c, n, dtype=F32))
    at = torch.arange(0, L, 61, device=DEV)
    rows = q[:, at, 0].double().reshape(Hq, d, -1)
    want = torch.stack([torch.softmax(r.T @ kr / d ** 0.5, 1) @ vr.T for r in rows])
    off = x[:, at, 0].double().reshape(Hq, d, -1).transpose(1, 2) / want - 1
    half, sums = (2.0 ** -11, 2.0 ** -12) if dtype == F16 else (2.0 ** -8, 2.0 ** -9)
    logits = 2.0 ** -13 if loud > 1 else 0
    assert off.abs().max().item() <= half + sums + logits, (off.abs().max().item(), off.mean().item())
    assert abs(off.mean().item()) <= sums + logits + 3 * half / 96 ** 0.5, off.mean().item()


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_short_histories_in_a_table_for_long_ones(dtype):
    """The same bits as with a table that just fits (blocks enough that keys are not cut into parts)."""
    gen = np.random.default_rng(37)
    d, H, L, cap, B, T = 16, 64, 45, 640, 2, 64
    c = _filled(gen, d * H, cap, B, H, T, "int8", True)
    q = _array(gen, (d * H, L, B), dtype)
    wide = nb.jl_empty(((1 << 20) // T, B), torch.int32, DEV)
    wide.fill_(-1)
    wide[:c.table.shape[0]] = c.t
    assert _path(c, q, H) == nb._lib.PATH_UMMA           # (also with the small table)
    for lens in ([640, 100], [45, 0]):
        want = nb.cached_attention(q, c.dev, _i32(lens), nheads=H, table=c.t, return_lse=True)
        got = nb.cached_attention(q, c.dev, _i32(lens), nheads=H, table=wide, return_lse=True)
        for g, w in zip(got, want):
            assert torch.equal(torch.nan_to_num(g, nan=7.0), torch.nan_to_num(w, nan=7.0))
    c.attend(q, [640, 100], H)


@gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("loud", [1, 64])
def test_sums_of_a_very_long_history_that_one_team_of_blocks_walks_over(dtype, code, loud):
    """Single queries of as many sequences as there are teams, so that a warp has a quarter of a history of 1048576 tokens;
    positive values.  Each addition of the products cuts off less than 2^-23 of the sum behind 16 keys, 2^-27 a key, and a warp
    adds 32768 keys that way: 2^-12; 2^-16 for all else (logits below 1, Float32 sums, weights' roundings that cancel over so
    many).  Rounding keeps order, so a result lies between the rounded ends of that range.  (Nothing is said of the mean of what
    is left: means of 1048576 values of a spread near 2 differ by 2 / 1024, less than a step, so their roundings are not
    independent, and 128 of them may be off by up to half a step together.)  ``loud``: the last third's logits are that much
    larger, so that maxima rise behind sums that have been put aside (sum |q||k| scale <= 8: 2 * 8 * 2^-18 = 2^-14 for weights)."""
    d, H, n, B = 16, 64, 1 << 20, 9
    gen = torch.Generator(device="cuda").manual_seed(8)
    c = nb.QuantizedCache(d * H, n, 1, nheads=H, page=64, eltype=CODE[code], device=DEV)
    lo, hi = ((-127, 128), (40, 128)) if code == "int8" else ((0x20, 0x58), (0x38, 0x50))     # (E4M3: 0.125 .. 15 and 1 .. 7.5)
    for t, (a, b) in ((c.k, lo), (c.v, hi)):
        (t if code == "int8" else t.view(torch.uint8)).random_(a, b, generator=gen)
    c.k_scale.fill_(2.0 ** -7 if code == "int8" else 2.0 ** -4)
    c.v_scale.fill_(2.0 ** -7 if code == "int8" else 2.0 ** -3)
    c.k_scale[:, n // 96:] *= loud
    t = nb.jl_empty((n // 64, B), torch.int32, DEV)
    t.copy_(torch.arange(n // 64, dtype=torch.int32, device=DEV)[:, None].expand(-1, B))
    q = (nb.jl_empty((d * H, 1, B), F32, DEV).normal_(generator=gen) * 2.0 ** -5).to(dtype)
    x = nb.cached_attention(q, c, n, nheads=H, table=t)
    off = 2.0 ** -12 + 2.0 ** -16 + (2.0 ** -14 if loud > 1 else 0)
    for h in range(0, H, 8):
        s = slice(h * d, (h + 1) * d)
        kr, vr = ((z[s].float() if code == "int8" else z[s].view(torch.uint8).contiguous().view(z.dtype).float()).double().permute(2, 1, 0).reshape(n, d)
                  * f[0].double().repeat_interleave(64)[:, None] for z, f in ((c.k, c.k_scale), (c.v, c.v_scale)))
        want = torch.softmax(q[s, 0].double().T @ kr.T / d ** 0.5, 1) @ vr                    # (B, d)
        got = x[s, 0].double().T
        low, high = ((want * (1 + e)).to(dtype).double() for e in (-off, off))
        assert (low <= got).all() and (got <= high).all(), ((got - low).min().item(), (high - got).min().item())


@gpu
def test_a_scale_that_is_none_in_float32():
    """1e-46 is 0 in Float32, which the C ABI takes for 1 / sqrt(d); the smallest number that is not is taken as it is."""
    gen = np.random.default_rng(39)
    d, H = 64, 2
    c = _filled(gen, d * H, 50, 1, H, 16, "int8", False)
    q = _array(gen, (d * H, 1, 1), F32)
    for scale in (1e-46, 1e-300, 0.0, -1e-46, 1e39):
        with pytest.raises(nb.ArgumentError):
            nb.cached_attention(q, c.dev, 50, nheads=H, scale=scale)
    x = nb.cached_attention(q, c.dev, 50, nheads=H, scale=1e-44)
    v = nb.cache_read(c.dev, 50, dtype=F32)[1].double()
    assert (x[:, 0].double() - v.mean(1)).abs().max().item() <= 2.0 ** -20 * v.abs().max().item()


@gpu
def test_a_caches_arrays_are_written_to_not_replaced():
    c = nb.QuantizedCache(32, 32, 2, nheads=2, page=16, device=DEV)
    for name in ("k", "v", "k_scale", "v_scale"):
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name).clone())
    with pytest.raises(AttributeError):
        c.batch = 1
    k = _array(np.random.default_rng(40), (32, 5, 2), F32)
    nb.cache_write_(c, k, k)
    before = nb.cache_read(c, 5, dtype=F32)[0]
    c.k_scale *= 2
    assert torch.equal(nb.cache_read(c, 5, dtype=F32)[0], 2 * before)


@gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_lengths_about_the_point_where_sums_are_put_aside(code):
    """256 tiles of 128 keys exactly, one key more, fewer, some more; queries on both sides of it; a poisoned page among the
    first, and a missing one that only the last queries see.  One table of pages for all sequences."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    d, H, L, n, T = 16, 16, 45, 33024, 64
    c = nb.QuantizedCache(d * H, n + T, 1, nheads=H, page=T, eltype=CODE[code], device=DEV)
    k, v = (nb.jl_empty((d * H, n + T, 1), F16, DEV).normal_(generator=gen) for _ in range(2))
    nb.cache_write_(c, k, v)
    c.v_scale[:, n // T] = NAN                                   # page 516, which no healthy sequence has
    lens = [32768, 32769, 32640, 33000, 5, 32790, 32800]
    B = len(lens)
    t = nb.jl_empty((n // T, B), torch.int32, DEV)
    t.copy_(torch.arange(n // T, dtype=torch.int32, device=DEV)[:, None].expand(-1, B))
    t[3, 5], t[512, 6] = n // T, -1                              # tokens 192 .. 255; 32768 .. 32831
    q = nb.jl_empty((d * H, L, B), F16, DEV).normal_(generator=gen)
    s = c._call(B, t)
    p = nb._lib.CacheAttnParams(dtype=nb._lib.F16, causal=1, Hq=H, L=L, q=0x1000, x=0x1000, lens=0x1000)
    lib = nb._lib.load()
    assert lib.nnlib_b200_cache_attn_path(C.byref(s), C.byref(p)) == nb._lib.PATH_UMMA
    assert lib.nnlib_b200_cache_attn_workspace_bytes(C.byref(s), C.byref(p)) >= 4 * d * H * L * B      # one part, with a row for sums
    x, lse = nb.cached_attention(q, c, _i32(lens), nheads=H, table=t, return_lse=True)
    nb.device_health()
    kr, vr = (z[:, :n, 0].double() for z in nb.cache_read(c, n, dtype=F32))
    for b, m in enumerate(lens):
        sees = torch.arange(n, device=DEV)[None] <= (m - L + torch.arange(L, device=DEV))[:, None]
        none = ~sees.any(1)
        bad = sees[:, 32768:32832].any(1) if b == 6 else torch.full((L,), b == 5, device=DEV)
        assert torch.equal(torch.isnan(x[:, :, b].float()).all(0), none | bad) and torch.equal(torch.isnan(x[:, :, b].float()).any(0), none | bad)
        assert torch.equal(torch.isneginf(lse[:, 0, b]), none)
        ok = ~(none | bad)
        if not ok.any():
            continue
        for h in range(H):
            r = slice(h * d, (h + 1) * d)
            logits = (q[r, ok, b].double().T @ kr[r] / d ** 0.5).masked_fill(~sees[ok], -INF)
            w = torch.softmax(logits, 1)
            want, size = w @ vr[r].T, w @ vr[r].abs().T
            lim = (2.0 ** -11 + 2.0 ** -13) * size + 2.0 ** -11 * want.abs() * 1.001 + 2.0 ** -25
            assert ((x[r, ok, b].double().T - want).abs() <= lim).all()
            torch.testing.assert_close(lse[ok, h, b].double(), torch.logsumexp(logits, 1), atol=2 * 12 * 2.0 ** -18, rtol=2.0 ** -20)
