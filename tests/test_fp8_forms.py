"""Which kernel an 8-bit product takes (host only), and what the queries refuse."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def cl():
    import cascadia_amd

    return cascadia_amd


@pytest.mark.parametrize("m,n,k,f32,tiles", [
    # sizes at which one side took at least 1.25 times the other's time
    (448, 4096, 1024, 0, True), (448, 4096, 1024, 1, True), (1024, 1900, 400, 0, True),
    (1024, 2395, 272, 1, True), (333, 7168, 576, 1, True), (512, 576, 7168, 0, True),
    (512, 576, 7168, 1, True), (512, 1137, 9152, 0, True), (800, 1137, 9152, 1, True),
    (333, 246, 4336, 0, False), (333, 246, 4336, 1, False), (17, 3037, 4992, 0, False),
    (200, 1137, 9152, 0, False), (160, 304, 4336, 1, False), (64, 2395, 272, 0, False)])
def test_the_faster_form(cl, m, n, k, f32, tiles):
    f = cl.lib().cascadia_int4_debug_fp8_gemm_form(n, k, 2, m, f32)
    assert f >= 3 if tiles else f == 2


def test_refusals(cl):
    arg, nul, L = cl._lib.ERR_ARG, cl._lib.ERR_NULL, cl.lib()
    f = L.cascadia_int4_debug_fp8_gemm_form
    for a in ((0, 64, 0, 4, 0), (32, 72, 0, 4, 0), (32, 64, 3, 4, 0), (32, 64, 0, 0, 0),
              (32, 64, 0, 4, 2)):
        assert f(*a) == arg
    f = L.cascadia_int4_debug_fp8_moe_form
    P = 1 << 20
    lay = cl._lib.Fp8MoeLayer(64, 32, 4, P, P, P, P, 0)
    assert f(None, 2, 4) == nul
    assert f(C.byref(lay), 0, 4) == arg and f(C.byref(lay), 2, 0) == arg
    assert [f(C.byref(lay), 2, t) for t in (1, 15, 16, 400)] == [0, 16, 128, 128]
