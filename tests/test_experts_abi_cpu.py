"""The C ABI of ragged groups of columns without a GPU: struct layouts, and argument checks that answer before any CUDA call."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np

from nnlib_jl_b200 import _lib
from oracle import experts_oracle as R

ROOT = Path(__file__).resolve().parent.parent


def test_struct_layouts_match_the_header(tmp_path):
    names = {"nnlib_b200_route_params": (_lib.RouteParams, ["G", "logits", "logits_stride", "bias", "weights", "position", "dweights", "dlogits"]),
             "nnlib_b200_grouped_params": (_lib.GroupedParams, ["zero_rest", "M", "R", "A", "strideA", "ldx", "C", "offsets", "columns", "status"]),
             "nnlib_b200_combine_params": (_lib.CombineParams, ["E", "k", "Y", "position", "y_stride", "columns", "dy_stride", "dY", "dweights"]),
             "nnlib_b200_adapter_params": (_lib.AdapterParams, ["transB", "M", "runs", "ldw", "strideA", "strideB", "ldx", "C", "run_len", "ids", "scale",
                                                                "scale0", "dC", "dX", "dA", "dB", "status"])}
    body = "".join(f'printf("%zu\\n", sizeof({t}));' + "".join(f'printf("%zu\\n", offsetof({t}, {f}));' for f in fields)
                   for t, (_, fields) in names.items())
    src = tmp_path / "sz.c"
    src.write_text('#include "nnlib_b200.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void){' + body + "return 0;}\n")
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-std=c99", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [n for t, fields in names.values() for n in [C.sizeof(t)] + [getattr(t, f).offset for f in fields]]


def _set(p, pointers, kw):
    for f in pointers:
        setattr(p, f, 0x1000)
    for f, v in kw.items():
        setattr(p, f, v)
    return C.byref(p)


def _route(**kw):
    return _set(_lib.RouteParams(dtype=_lib.F32, normalize=1, G=16, N=10, k=2),
                ("logits", "weights", "experts", "offsets", "columns", "position", "dweights", "dlogits"), kw)


def _grouped(**kw):
    return _set(_lib.GroupedParams(dtype=_lib.BF16, M=32, K=16, G=3, N=10, R=10, lda=32, strideA=512, ldx=16, ldc=32), ("A", "X", "C", "offsets"), kw)


def _combine(**kw):
    return _set(_lib.CombineParams(dtype=_lib.BF16, E=8, N=5, R=10, k=2), ("Y", "position", "weights", "y", "columns", "dy", "dY", "dweights"), kw)


def _adapter(**kw):
    return _set(_lib.AdapterParams(dtype=_lib.F32, M=32, K=16, N=10, r=4, n=2, runs=2, ldw=32, lda=4, strideA=64, ldb=32, strideB=128, ldx=16, ldc=32,
                                   run_len=5, scale0=1.0, lddc=32), ("W", "A", "B", "X", "C", "ids", "dC", "dX", "dA", "dB"), kw)


def test_router_argument_checks_without_a_gpu(lib):
    fwd = lambda **kw: lib.nnlib_b200_route(_route(**kw), None, 0, None)
    bwd = lambda **kw: lib.nnlib_b200_route_bwd(_route(**kw), None)
    for bad in (dict(struct_size=8), dict(dtype=3), dict(G=0), dict(N=-1), dict(k=0), dict(k=17), dict(logits_stride=15), dict(logits=None),
                dict(weights=None), dict(experts=None), dict(logits=0x1002), dict(weights=0x1002), dict(N=2 ** 30 + 1)):
        assert fwd(**bad) == bwd(**bad) == _lib.INVALID_ARG, bad
    for bad in (dict(offsets=None), dict(columns=None), dict(position=None), dict(bias=0x1001)):
        assert fwd(**bad) == _lib.INVALID_ARG, bad
    for bad in (dict(dweights=None), dict(dlogits=None)):
        assert bwd(**bad) == _lib.INVALID_ARG, bad
    assert fwd(G=1025) == fwd(G=64, k=33) == _lib.UNSUPPORTED_SHAPE
    assert bwd(N=0) == _lib.OK
    # few tokens are one block's; more leave counts
    need = lambda **kw: lib.nnlib_b200_route_workspace_bytes(_route(**kw))
    assert need() == need(N=128) == 0 and need(N=5000) > 0 and need(k=0, N=5000) == 0
    assert fwd(N=5000) == _lib.WORKSPACE_TOO_SMALL
    assert lib.nnlib_b200_route(_route(N=5000), 0x1008, 1 << 20, None) == _lib.WORKSPACE_TOO_SMALL


def test_grouped_argument_checks_without_a_gpu(lib):
    big = 1 << 40
    calls = lambda **kw: tuple(f(_grouped(**kw), 0x1000, big, None) for f in (lib.nnlib_b200_grouped_gemm, lib.nnlib_b200_grouped_gemm_grad))
    for bad in (dict(struct_size=8), dict(dtype=3), dict(M=-1), dict(K=-1), dict(N=-1), dict(R=-1), dict(G=-1), dict(lda=31), dict(strideA=-1), dict(ldx=15),
                dict(ldc=31), dict(A=None), dict(X=None), dict(C=None), dict(offsets=None), dict(A=0x1001), dict(offsets=0x1002), dict(columns=0x1001),
                dict(R=11), dict(transA=1, lda=15), dict(status=0x1001), dict(M=2 ** 31)):
        assert calls(**bad) == (_lib.INVALID_ARG,) * 2, bad
    assert calls(G=40000) == (_lib.UNSUPPORTED_SHAPE,) * 2
    before = lib.nnlib_b200_launch_count()
    assert calls(M=0) == (_lib.OK,) * 2 and calls(R=0)[0] == _lib.OK and calls(K=0)[1] == _lib.OK and calls(G=0)[1] == _lib.OK
    assert lib.nnlib_b200_launch_count() == before


def test_combine_argument_checks_without_a_gpu(lib):
    fwd = lambda **kw: lib.nnlib_b200_combine(_combine(**kw), None)
    bwd = lambda **kw: lib.nnlib_b200_combine_bwd(_combine(**kw), None)
    for bad in (dict(struct_size=8), dict(dtype=3), dict(E=0), dict(N=-1), dict(R=-1), dict(k=0), dict(Y=None), dict(position=None), dict(Y=0x1001),
                dict(position=0x1002), dict(Y_stride=7), dict(dy_stride=7), dict(N=2 ** 31 - 1)):
        assert fwd(**bad) == bwd(**bad) == _lib.INVALID_ARG, bad
    assert fwd(y=None) == bwd(dy=None) == bwd(dY=None) == bwd(columns=None) == _lib.INVALID_ARG
    assert fwd(k=33) == _lib.UNSUPPORTED_SHAPE and fwd(N=0) == bwd(N=0, R=0) == _lib.OK


def test_adapter_argument_checks_without_a_gpu(lib):
    big = 1 << 40
    fwd = lambda **kw: lib.nnlib_b200_adapter_gemm(_adapter(**kw), 0x1000, big, None)
    bwd = lambda **kw: lib.nnlib_b200_adapter_bwd(_adapter(**kw), 0x1000, big, None)
    for bad in (dict(struct_size=8), dict(dtype=3), dict(M=-1), dict(K=-1), dict(N=-1), dict(r=0), dict(n=-1), dict(runs=-1), dict(run_len=-1), dict(ldw=31),
                dict(lda=3), dict(ldb=31), dict(strideA=-1), dict(W=None), dict(A=None), dict(B=None), dict(ids=None), dict(W=0x1002), dict(ids=0x1002),
                dict(offsets=0x1002), dict(scale=0x1001), dict(transA=1, lda=15)):
        assert fwd(**bad) == bwd(**bad) == _lib.INVALID_ARG, bad
    assert fwd(X=None) == fwd(C=None) == fwd(ldx=15) == bwd(dC=None) == bwd(dX=None) == bwd(dA=None) == bwd(lddc=31) == _lib.INVALID_ARG
    assert fwd(r=129, lda=129) == bwd(runs=2 ** 21) == _lib.UNSUPPORTED_SHAPE
    need = lib.nnlib_b200_adapter_gemm_workspace_bytes(_adapter())
    assert need > 0 and lib.nnlib_b200_adapter_gemm(_adapter(), 0x1000, need - 1, None) == _lib.WORKSPACE_TOO_SMALL
    assert lib.nnlib_b200_adapter_bwd(_adapter(), None, big, None) == _lib.WORKSPACE_TOO_SMALL
    assert fwd(N=0) == _lib.OK


def test_the_oracles_gradients_are_those_of_differences():
    gen = np.random.default_rng(0)
    step = 1e-6

    def check(f, args, grads):
        for i, (v, g) in enumerate(zip(args, grads)):
            u = gen.standard_normal(v.shape)
            moved = [[a + s * u if j == i else a for j, a in enumerate(args)] for s in (step, -step)]
            assert abs((f(*moved[0]) - f(*moved[1])) / (2 * step) - (g * u).sum()) < 1e-6 * (1 + abs(g).sum())

    x, dw = gen.standard_normal((6, 9)), gen.standard_normal((2, 9))
    for normalize in (True, False):
        e = R.route(x, 2, normalize=normalize)[1]
        check(lambda v: (R.route(v, 2, normalize=normalize)[0] * dw).sum(), [x], [R.route_back(x, e, dw, normalize)])
    A, X, dC, o, c = gen.standard_normal((5, 7, 3)), gen.standard_normal((7, 6)), gen.standard_normal((5, 8)), [0, 3, 3, 7], [1, 1, 5, 0, 9, 2, -1, 3]
    check(lambda a, x: (R.grouped(a, x, o, c) * dC).sum(), [A, X], R.grouped_back(A, X, o, dC, c))
    Y, p, w, dy = gen.standard_normal((4, 8)), np.array([[0, 3, -1], [7, 2, 1]]), gen.standard_normal((2, 3)), gen.standard_normal((4, 3))
    check(lambda y, v: (R.combine(y, p, v) * dy).sum(), [Y, w], R.combine_back(Y, p, w, dy))
    W, A, B, X, dY = (gen.standard_normal(s) for s in ((5, 7), (3, 7, 2), (5, 3, 2), (7, 9), (5, 9)))
    ids, o, s = [1, 0, 1, 4], [0, 2, 2, 7, 8], np.array([0.5, 2.0])
    check(lambda x, a, b: (R.adapters(W, x, a, b, ids, o, s) * dY).sum(), [X, A, B], R.adapters_back(W, X, A, B, ids, o, s, dY))
