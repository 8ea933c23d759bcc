"""Sizes past what one launch takes (fewer than 2^32 threads along a grid's dimension)
are refused as arguments, on the CPU: no call here reaches the device."""
import ctypes as C

import pytest

P = 1 << 20  # an address that no call may read


@pytest.fixture(scope="module")
def cl():
    import cascadia_amd

    return cascadia_amd


def test_route(cl):
    r = cl._lib.Router(n_experts=1, top_k=1, score=1, n_groups=1, top_groups=1, group_best=1,
                       normalize=1, scale=1.0, bias=None)
    f = cl.lib().cascadia_int4_route_experts
    for t in ((1 << 25) + 1, 1 << 26, 1 << 30):
        assert f(C.byref(r), P, 0, t, P, P, None) == cl._lib.ERR_ARG


def test_quantize(cl):
    f = cl.lib().cascadia_int4_fp8_quantize
    for rows, k in ((1 << 24, 2048), (1 << 24, 1 << 20), (1 << 21, 16384), (1 << 15, 1 << 20)):
        assert f(P, 0, rows, k, P, P, None) == cl._lib.ERR_ARG, (rows, k)


def test_product(cl):
    L = cl.lib()
    for xt in (0, 2):
        for n, k, m in ((16, 2048, 1 << 24), (1 << 24, 128, 1 << 14), (1 << 24, 16, 1 << 24)):
            a = (n, k, P, P, P, xt, P if xt == 2 else None, m, P, 0, None, None)
            assert L.cascadia_int4_fp8_gemm(*a) == cl._lib.ERR_ARG, (n, k, m)
            assert L.cascadia_int4_fp8_gemm_workspace_bytes(n, k, xt, m) == 0
            assert L.cascadia_int4_debug_fp8_gemm_form(n, k, xt, m, 0) == cl._lib.ERR_ARG
        # (the most rows of a narrow product stay)
        assert L.cascadia_int4_fp8_gemm_workspace_bytes(16, 128, xt, 1 << 24) > 0


def test_tiling(cl):
    f = cl.lib().cascadia_int4_fp8_tile_weights
    for a in ((1 << 20, 16 * 128, 128), (1, 1 << 24, 128 << 7), (1 << 17, 128, 128 * 128)):
        assert f(*a, P, P, None) == cl._lib.ERR_ARG, a


def test_layer(cl):
    L, Layer = cl.lib(), cl._lib.Fp8MoeLayer

    def call(hidden, inter, experts, k, t):
        lay = Layer(hidden, inter, experts, P, P, P, P, 0)
        size = L.cascadia_int4_fp8_moe_workspace_bytes(C.byref(lay), k, t)
        if size:  # accepted: nothing is launched here
            return 0
        return L.cascadia_int4_fp8_moe_forward(C.byref(lay), k, P, P, 0.0, P, 0, None, t, P, 0,
                                               None, None)

    arg = cl._lib.ERR_ARG
    assert call(16, 1 << 20, 1024, 16, 500) == arg      # chunks of 16 rows, a wide inter
    assert call(1 << 20, 16, 1024, 16, 500) == arg      # a wide hidden
    assert call(16, 1 << 16, 1, 16, 1 << 20) == arg     # tiles
    assert call(1 << 11, 16, 1, 16, 1 << 20) == arg     # n_tokens * hidden
    for a in ((7168, 2048, 384, 8, 1), (7168, 2048, 384, 8, 16384), (4096, 14336, 8, 2, 65536),
              (16, 16, 1024, 16, 1 << 20), (16, 16, 1, 1, 1 << 20)):
        assert call(*a) == 0, a
