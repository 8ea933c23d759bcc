"""Which kernel an 8-bit product takes (host only): every form is reached by sizes of
the GPU tests, and what the queries refuse."""
import ctypes as C

import pytest

from test_gpu_fp8 import GEMM_SIZES
from test_gpu_fp8_tiles import SIZES, F32


@pytest.fixture(scope="module")
def cl():
    import cascadia_amd

    return cascadia_amd


def test_sizes_of_the_gpu_tests_take_every_form(cl):
    f = cl.lib().cascadia_int4_debug_fp8_gemm_form
    for want, m, n, k, dtype in SIZES:
        assert f(n, k, 2, m, int(dtype == F32)) == want, (m, n, k)
    # both output types of every tile form but the largest, which f32 does not take
    assert {(w, d == F32) for w, _, _, _, d in SIZES} == {
        (w, f32) for w in (3, 4, 5, 6) for f32 in (False, True) if w < 6 or not f32}
    assert {f(n, k, t, m, 0) for m, n, k in GEMM_SIZES for t in (0, 2)} >= {0, 1, 2}


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
