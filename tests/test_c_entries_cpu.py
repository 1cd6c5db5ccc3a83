"""Refusals of the C entries of RMSNorm and the 8-bit products (host checks: pointer values are never dereferenced, nothing is launched)."""
import ctypes as C

import pytest

ARG, SHAPE, WS = -1, -2, -3
ONE, ODD, OFF8 = C.c_void_p(4096), C.c_void_p(4097), C.c_void_p(4096 + 8)


@pytest.fixture(scope="module")
def L():
    from spn4cir_amd import _lib
    return _lib.lib()


def test_rmsnorm_alignment_and_types(L):
    """Blocks start at 8 bytes, a workspace at 16; the second copy of dx has a type of its own, looked at only where it is wanted."""
    fwd = lambda y, yt, ys: L.spn_rmsnorm_fwd(ONE, 1, 64, None, 0, 0, ONE, 1e-6, None, y, yt, ys, ONE, 2, 64, None)  # noqa: E731
    assert fwd(ODD, 3, ONE) == ARG and fwd(C.c_void_p(4096 + 4), 3, ONE) == ARG
    bwd = lambda rows, ws, nb, dx2=None, d2=0: L.spn_rmsnorm_bwd(ONE, 1, 64, ONE, 1, 64, ONE, ONE, None, 0, ONE, dx2, d2, ONE, rows, 64, ws, nb, None)  # noqa: E731,E501
    need = L.spn_rmsnorm_bwd_workspace_bytes(5000, 64)
    assert need > 0 and bwd(5000, OFF8, need) == WS and bwd(5000, ODD, need) == WS and bwd(5000, ONE, need - 1) == WS
    assert bwd(5000, ONE, need, ONE, 3) == ARG and bwd(5000, ONE, need, ONE, -1) == ARG and bwd(5000, ONE, need, ONE, 7) == ARG
    assert bwd(5000, ODD, need, None, 7) == WS                       # (no second copy: its type is not looked at)


def test_product_workspace(L):
    """Where k slices need one: not NULL, large enough, 16-byte aligned."""
    g = lambda ws, nb: L.spn_gemm_nt_fp8(ONE, ONE, ONE, ONE, 2304, 768, 19712, None, 0, ONE, 1, 768, 0, ws, nb, None)  # noqa: E731
    need = L.spn_gemm_nt_fp8_workspace_bytes(2304, 768, 19712)
    assert need > 0 and g(None, need) == WS and g(ONE, need - 1) == WS and g(OFF8, need) == WS and g(None, 0) == WS


def test_pitch_of_scale_bytes(L):
    """Blocks that are quantised again: a row of scale bytes holds one for each block."""
    for C_, pitch in ((128, 0), (129, 1), (1000, 7)):
        assert L.spn_quantize_fp8(ONE, 3, 1024, ONE, pitch, 4, C_, 0, None, None, ONE, ONE, None, None, 0, None) == SHAPE
