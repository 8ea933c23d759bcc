"""Every form of the 8-bit products on tiles: ragged sizes that the rule sends there,
both output types, more blocks of K than the scales' two windows hold, against the
64-bit reference (fp8_ref).  Each test asserts the form that its sizes take, so that a
change of the rule cannot take the kernels out of it unseen."""
import ctypes as C

import numpy as np
import pytest
import torch

import fp8_ref as ref
from test_gpu_fp8 import cl, eight_bit, gemm_case, gemm_ref, gen, moe_case, moe_ref, run_moe  # noqa: F401

pytestmark = pytest.mark.gpu

ROWS32, TILES, SLICES, WIDE, LARGE = 2, 3, 4, 5, 6
F32, BF16 = torch.float32, torch.bfloat16

# (form, rows, n, k, output)
SIZES = [
    (SLICES, 17, 320, 9232, F32), (SLICES, 65, 576, 9232, BF16), (SLICES, 65, 576, 9232, F32),
    (SLICES, 300, 321, 12304, BF16), (SLICES, 129, 130, 9360, F32), (SLICES, 40, 31, 9232, BF16),
    (SLICES, 100, 4100, 4112, F32), (SLICES, 333, 1500, 4112, BF16), (TILES, 448, 4096, 1024, BF16),
    (TILES, 2000, 1900, 400, BF16), (TILES, 2000, 1900, 400, F32),
    (TILES, 1900, 2001, 1552, BF16), (TILES, 1905, 1999, 1680, F32),
    (WIDE, 1700, 3600, 1168, BF16), (WIDE, 1700, 3601, 1296, F32), (WIDE, 2305, 2304, 1680, BF16),
    (WIDE, 3500, 3600, 1168, F32), (WIDE, 4100, 4200, 1296, F32),
    (LARGE, 3500, 3600, 1168, BF16), (LARGE, 4100, 4200, 1296, BF16), (LARGE, 4097, 3585, 1680, BF16)]


def form(cl, m, n, k, dtype, x_type=2):
    return cl.lib().cascadia_int4_debug_fp8_gemm_form(n, k, x_type, m, int(dtype == F32))


def wide_scales(g, *shape):
    return 2.0 ** torch.randint(-12, 13, shape, generator=g).float()


def case(seed, m, n, k):
    """Codes whose blocks' scales are powers of two far apart: one block's taken for
    another's is far off."""
    w, ws, x, xs = gemm_case(seed, m, n, k, "fp8")
    g = gen(seed + 1)
    return w, wide_scales(g, *ws.shape), x, wide_scales(g, *xs.shape)


def run(cl, w, ws, x, xs, y, workspace=None):
    m, k = x.shape
    return cl.fp8_gemm(w, ws, x, w.shape[0], k, m, y, x_scales=xs, workspace=workspace)


def rows_of(m):
    return sorted({0, 1, m // 2, m - 2, m - 1} | {r for r in (31, 127, 128, 255, 256) if r < m}
                  | set(range(77, m, 997)))


@pytest.mark.parametrize("f,m,n,k,dtype", SIZES)
def test_every_form(cl, f, m, n, k, dtype):
    assert form(cl, m, n, k, dtype) == f
    w, ws, x, xs = case(m + n, m, n, k)
    d = [t.cuda() for t in (w, ws, x, xs)]
    y = run(cl, *d, torch.full((m, n), float("nan"), dtype=dtype, device="cuda"))
    assert torch.isfinite(y).all()
    for _ in range(2):  # and the same again
        assert torch.equal(run(cl, *d, torch.empty_like(y)), y)
    rows = rows_of(m)
    got = y[rows].double().cpu().numpy()
    for i, r in enumerate(rows):
        want, bound = gemm_ref(w, ws, x[r:r + 1], xs[r:r + 1])
        if dtype == BF16:
            bound = bound + eight_bit(w, ws, x[r:r + 1], xs[r:r + 1])
            bound = bound + ref.BF16 * (np.abs(want) + bound)
        assert np.all(np.abs(got[i] - want[0]) <= bound[0]), r


@pytest.mark.parametrize("f,m,n,k", [(SLICES, 130, 254, 9232), (TILES, 2000, 1900, 400),
                                     (WIDE, 18500, 254, 256), (LARGE, 33000, 254, 256)])
def test_every_code_in_8_bit_sums(cl, f, m, n, k):
    """Every finite code, subnormal ones among them, times one, anywhere in a row of
    zeros: exact, and held exactly by bf16."""
    assert form(cl, m, n, k, BF16) == f
    finite = torch.tensor([c for c in range(256) if c & 0x7F != 0x7F], dtype=torch.uint8)
    code = finite[torch.arange(n) % 254]
    w = torch.zeros((n, k), dtype=torch.uint8)
    w[torch.arange(n), torch.randint(0, k, (n,), generator=gen(m))] = code
    x = torch.ones((m, k), device="cuda").to(torch.float8_e4m3fn)
    one = torch.ones
    y = torch.empty((m, n), dtype=BF16, device="cuda")
    run(cl, w.cuda(), one((ref.blocks(n), ref.blocks(k)), device="cuda"), x,
        one((m, ref.blocks(k)), device="cuda"), y)
    want = code.view(torch.float8_e4m3fn).to(BF16).cuda()
    assert torch.equal(y, want.expand(m, n))


@pytest.mark.parametrize("f,m,n,k,dtype", [
    (SLICES, 65, 576, 9232, BF16), (SLICES, 65, 576, 9232, F32), (TILES, 2000, 1900, 400, BF16),
    (TILES, 2000, 1900, 400, F32), (WIDE, 1700, 3600, 208, BF16), (WIDE, 1700, 3600, 208, F32),
    (LARGE, 3500, 3600, 208, BF16)])
def test_nan_stays_in_its_row(cl, f, m, n, k, dtype):
    assert form(cl, m, n, k, dtype) == f
    w, ws, x, xs = gemm_case(1, m, n, k, "fp8")
    x.view(torch.uint8)[m - 1, k - 1] = 0x7F
    x.view(torch.uint8)[3, 130] = 0xFF
    w.view(torch.uint8)[n - 3, 0] = 0xFF
    y = run(cl, *(t.cuda() for t in (w, ws, x, xs)), torch.empty((m, n), dtype=dtype, device="cuda"))
    want = torch.zeros((m, n), dtype=torch.bool)
    want[m - 1], want[3], want[:, n - 3] = True, True, True
    assert torch.equal(torch.isnan(y).cpu(), want)


@pytest.mark.parametrize("f,m,n,k,dtype", [
    (SLICES, 65, 577, 9232, BF16), (SLICES, 65, 577, 9232, F32), (SLICES, 65, 576, 9232, BF16),
    (SLICES, 65, 576, 9232, F32), (TILES, 2000, 1900, 400, BF16), (TILES, 2000, 1900, 400, F32),
    (WIDE, 1700, 3601, 208, BF16), (WIDE, 1700, 3600, 208, F32), (LARGE, 3500, 3600, 208, BF16),
    (LARGE, 3500, 3597, 208, BF16)])
def test_writes_its_rows_only_at_any_alignment(cl, f, m, n, k, dtype):
    assert form(cl, m, n, k, dtype) == f
    d = [t.cuda() for t in gemm_case(2, m, n, k, "fp8")]
    want = run(cl, *d, torch.empty((m, n), dtype=dtype, device="cuda"))
    for at in (64, 65):
        buf = torch.full((m * n + 128,), 3.0, dtype=dtype, device="cuda")
        run(cl, *d, buf[at:at + m * n])
        assert torch.equal(buf[at:at + m * n].view(m, n), want)
        assert torch.all(buf[:at] == 3.0) and torch.all(buf[at + m * n:] == 3.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["fp8", "bf16", "f32"])
def test_one_workspace_serves_smaller_calls(cl, kind, dtype):
    """Slices of K joined in a caller's workspace, sized for the most rows."""
    n, k, most = 320, 12304, 400
    w, ws, x, xs = (None if t is None else t.cuda() for t in gemm_case(8, most, n, k, kind))
    need = cl.fp8_gemm_workspace_bytes(n, k, most, x.dtype)
    buf = torch.full((need + 256,), 0xA5, dtype=torch.uint8, device="cuda")
    for m in (400, 300, 129, 128, 65, 33, 17, 16, 1):
        if m > 16:
            assert form(cl, m, n, k, dtype) == SLICES
        sc = None if xs is None else xs[:m].contiguous()
        a = run(cl, w, ws, x[:m], sc, torch.empty((m, n), dtype=dtype, device="cuda"), buf[:need])
        b = run(cl, w, ws, x[:m], sc, torch.empty((m, n), dtype=dtype, device="cuda"))
        assert torch.equal(a, b)
    assert torch.all(buf[need:] == 0xA5)


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("T,H,I,E,k", [(40, 1168, 144, 3, 2), (70, 1296, 1168, 1, 1),
                                       (150, 1168, 272, 2, 2), (16, 2064, 1040, 2, 1)])
def test_layer_of_many_blocks(cl, T, H, I, E, k, out_dtype):
    """Experts on tiles over more blocks than the scales' windows hold, their scales
    powers of two apart, codes as given and in blocks."""
    lay = cl._lib.Fp8MoeLayer(H, I, E, 256, 256, 256, 256, 0)
    assert cl.lib().cascadia_int4_debug_fp8_moe_form(C.byref(lay), k, T) == 128
    c = list(moe_case(T + H, T, H, I, E, k, BF16))
    g = gen(T)
    for i in (1, 3):
        c[i] = c[i] * 2.0 ** torch.randint(-2, 3, c[i].shape, generator=g).float()
    res = c[-1].to(out_dtype)
    want, bound = moe_ref(c, 0.0, res)
    if out_dtype == BF16:
        bound = bound + ref.BF16 * (np.abs(want) + bound)
    outs = [run_moe(cl, c, out_dtype, 0.0, res, tiled=t) for t in (True, False)]
    assert torch.equal(*outs)
    assert np.all(np.abs(outs[0].double().cpu().numpy() - want) <= bound)
