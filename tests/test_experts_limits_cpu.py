"""Sizes that the C ABI of ragged groups of columns refuses before any CUDA call: the kernels count a tile beyond an extent in 32 bits."""
import pytest

from nnlib_jl_b200 import _lib
from test_experts_abi_cpu import _adapter, _combine, _grouped, _route

NEAR = 2 ** 31 - 1
BIG = 1 << 62


@pytest.mark.parametrize("n", [NEAR, NEAR - 128, NEAR - 65535])
def test_extents_near_what_32_bits_count(lib, n):
    wide = dict(lda=n, ldx=n, ldc=n, strideA=2 * n)
    for f in (lib.nnlib_b200_grouped_gemm, lib.nnlib_b200_grouped_gemm_grad):
        for kw in (dict(M=n), dict(K=n), dict(N=n), dict(N=n, R=n)):
            assert f(_grouped(**wide, **kw), 0x1000, BIG, None) == _lib.UNSUPPORTED_SHAPE, kw
    wide = dict(ldw=n, lda=n, ldb=n, ldx=n, ldc=n, lddc=n, strideA=2 * n, strideB=2 * n)
    for f in (lib.nnlib_b200_adapter_gemm, lib.nnlib_b200_adapter_bwd):
        for kw in (dict(M=n), dict(K=n), dict(N=n)):
            assert f(_adapter(**wide, **kw), 0x1000, BIG, None) == _lib.UNSUPPORTED_SHAPE, kw
    for f in (lib.nnlib_b200_combine, lib.nnlib_b200_combine_bwd):
        assert f(_combine(E=n), None) == _lib.UNSUPPORTED_SHAPE
        assert f(_combine(R=n), None) == (_lib.INVALID_ARG if n > NEAR - 8 else _lib.UNSUPPORTED_SHAPE)
    assert lib.nnlib_b200_route(_route(N=n, k=1), 0x1000, BIG, None) == lib.nnlib_b200_route_bwd(_route(N=n, k=1), None) == _lib.UNSUPPORTED_SHAPE
    assert lib.nnlib_b200_route_workspace_bytes(_route(N=n, k=1)) == 0


def test_gradients_that_would_be_written_to_one_matrix(lib):
    """strideA = 0: one matrix for all runs is read, not written."""
    f = lambda **kw: lib.nnlib_b200_grouped_gemm_grad(_grouped(strideA=0, **kw), 0x1000, BIG, None)
    assert f() == _lib.INVALID_ARG and f(M=0) == _lib.OK
