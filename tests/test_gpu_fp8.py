"""Routing to experts and the 8-bit floating-point products on the GPU, each
against a 64-bit reference (fp8_ref) with bounds that count its roundings."""
import numpy as np
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def cl():
    import cascadia_amd

    return cascadia_amd


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g).to(dtype)


def codes(g, *shape):
    return (torch.randn(shape, generator=g) * 112).clamp_(-448, 448).to(FP8)


def scales(g, *shape):
    return torch.rand(shape, generator=g) * 0.02 + 0.005


# ---------------------------------------------------------------------------
# routing
# ---------------------------------------------------------------------------

def run_route(cl, logits, top_k, score, bias, groups, top_groups, best, norm, scale):
    T = logits.shape[0]
    ids = torch.full((T, top_k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((T, top_k), float("nan"), device="cuda")
    cl.route_experts(logits.cuda(), top_k, ids, w,
                     score=cl.SCORE_SIGMOID if score == "sigmoid" else cl.SCORE_SOFTMAX,
                     bias=None if bias is None else bias.cuda(), n_groups=groups,
                     top_groups=top_groups, group_best=best, normalize=norm, scale=scale)
    return ids.cpu().numpy(), w.cpu().numpy()


def check_route(cl, logits, top_k, score, bias, groups, top_groups, best, norm, scale):
    ids, w = run_route(cl, logits, top_k, score, bias, groups, top_groups, best, norm, scale)
    rid, rw = ref.route(logits.double().numpy(), top_k, score,
                        None if bias is None else bias.numpy(), groups, top_groups, best, norm,
                        scale)
    assert np.array_equal(ids, rid)
    # s rounds once to f32; sum, division and scale: top_k + 3 roundings
    assert np.all(np.abs(w - rw) <= (top_k + 6) * ref.U32 * np.abs(rw) + 1e-37)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,groups,top_groups,best,bias,norm", [
    (1, 256, 8, 8, 4, 2, True, True), (1, 1, 1, 1, 1, 1, False, True),
    (5, 60, 4, 1, 1, 1, False, False), (33, 64, 16, 1, 1, 2, True, True),
    (7, 65, 3, 5, 2, 2, True, False), (130, 384, 8, 1, 1, 1, True, True),
    (3, 1024, 16, 64, 1, 1, False, True), (2, 1023, 6, 3, 3, 2, True, True),
    (4, 32, 2, 32, 2, 2, False, True), (9, 160, 6, 8, 3, 1, True, False),
    (257, 128, 8, 4, 2, 2, False, True), (2, 16, 16, 4, 4, 2, True, True),
    (66, 500, 1, 2, 1, 2, True, True), (3, 4, 2, 1, 1, 1, True, True)])
def test_route_matches_the_definition(cl, dtype, score, T, E, k, groups, top_groups, best, bias,
                                      norm):
    g = gen(T * 1000 + E)
    logits = (normal(g, T, E) * 2).to(dtype)
    b = normal(g, E) * 0.1 if bias else None
    check_route(cl, logits, k, score, b, groups, top_groups, best, norm, 2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (8, 3)])
def test_route_ties_go_to_the_lower_id(cl, score, groups, top_groups):
    g = gen(3)
    logits = torch.randint(-2, 3, (70, 96), generator=g).float()
    check_route(cl, logits, 8, score, None, groups, top_groups, 2, True, 1.0)
    bias = torch.zeros(96)
    check_route(cl, logits, 8, score, bias, groups, top_groups, 1, True, 1.0)
    check_route(cl, torch.zeros(2, 96), 16, score, None, groups, top_groups, 1, True, 1.0)


def test_route_close_scores(cl):
    """Scores that 32 bits do not tell apart: sigmoids of logits one f32 step
    apart, and biases that almost cancel the difference."""
    g = gen(4)
    base = normal(g, 200, 1) * 2
    step = torch.randint(0, 6, (200, 64), generator=g).float()
    logits = base + step * 2.0 ** -22
    bias = torch.randint(-3, 4, (64,), generator=g).float() * 2.0 ** -25
    for b in (None, bias):
        check_route(cl, logits, 8, "sigmoid", b, 1, 1, 1, True, 1.0)
        check_route(cl, logits, 8, "softmax", b, 8, 4, 2, False, 1.0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
def test_route_infinities_and_nan(cl, score, groups, top_groups):
    inf, nan = float("inf"), float("nan")
    g = gen(5)
    x = normal(g, 9, 48)
    x[0, 5:] = -inf                        # fewer left than are chosen
    x[1] = -inf                            # nothing left
    x[2, 3] = nan
    x[3, ::2] = nan
    x[4, 7] = inf
    x[5, 7], x[5, 40] = inf, inf
    x[6] = nan
    x[7] = torch.finfo(torch.float32).min  # masked by the lowest value
    x[8, 1:] = torch.finfo(torch.float32).min
    check_route(cl, x, 6, score, None, groups, top_groups, 2, True, 2.0)
    check_route(cl, x, 6, score, None, groups, top_groups, 1, False, 2.0)
    check_route(cl, x, 6, score, normal(g, 48) * 0.1, groups, top_groups, 1, True, 2.0)


def test_route_groups_whose_biases_cancel(cl):
    """A group's best two, of opposite signs and far larger than their sum: added in
    32 bits that sum would be off by 2^-24 of them, more than groups are apart."""
    g = torch.Generator().manual_seed(18)
    logits = torch.randn((512, 16), generator=g)
    for big in (30.0, 1000.0, 65536.0):
        bias = torch.tensor([big, -big] * 8)
        check_route(cl, logits, 4, "sigmoid", bias, 8, 3, 2, True, 1.0)
        check_route(cl, logits, 4, "softmax", bias, 8, 3, 2, True, 1.0)


def test_route_nothing_and_refusals(cl):
    ids = torch.empty((0, 2), dtype=torch.int32, device="cuda")
    w = torch.empty((0, 2), device="cuda")
    cl.route_experts(torch.empty((0, 8), device="cuda"), 2, ids, w)
    x = torch.zeros((3, 8), device="cuda")
    ids = torch.empty((3, 2), dtype=torch.int32, device="cuda")
    w = torch.empty((3, 2), device="cuda")
    for kw in ({"n_groups": 3}, {"n_groups": 0}, {"n_groups": 4, "top_groups": 5},
               {"group_best": 3}, {"score": 2}, {"bias": torch.zeros(7, device="cuda")},
               {"bias": torch.zeros(8)}, {"n_groups": 8, "top_groups": 1}):
        with pytest.raises(ValueError):
            cl.route_experts(x, 2, ids, w, **kw)
    for a in ((x.half(), 2, ids, w), (x.t(), 2, ids, w), (x, 3, ids, w), (x, 2, ids.long(), w),
              (x.cpu(), 2, ids, w), (x, 2, ids, w.double()), (x.view(-1), 2, ids, w)):
        with pytest.raises(ValueError):
            cl.route_experts(*a)


# ---------------------------------------------------------------------------
# quantisation
# ---------------------------------------------------------------------------

def check_codes(got, x, rows, exact):
    """Codes are the quotients' rounding (bf16 values: exactly, f32 values: a
    nearest one but for a quotient within its own rounding of the border)."""
    q, s = ref.quotients(x, rows)
    c, sc = got
    assert np.array_equal(sc, (ref.tops(np.asarray(x, np.float64), rows).astype(np.float32)
                               / np.float32(448)))
    if exact:
        assert np.array_equal(c, ref.round_e4m3(q))
    else:
        assert np.all(np.abs(c - q) <= ref.e4m3_step(q) / 2 + 4 * ref.U32 * np.abs(q))


def quantize(cl, x):
    r, k = x.shape
    c = torch.full((r, k), 0x7F, dtype=torch.uint8, device="cuda")
    s = torch.full((r, ref.blocks(k)), float("nan"), device="cuda")
    cl.quantize_fp8(x.cuda(), r, k, c, s)
    return ref.e4m3(c), s.cpu().numpy()


def spread_values(g, r, k, dtype):
    """Normal values of groups from 2^-110 to 2^100, wide ones, zeros."""
    x = normal(g, r, k)
    x *= 2.0 ** torch.randint(-20, 20, (r, 1), generator=g).float()
    x[:, ::17] *= 30
    x[:, 5::23] = 0
    x[:1] *= 2.0 ** -100
    if r > 2:
        x[1] = 0
        x[2] *= 2.0 ** 70
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("r,k", [(1, 16), (1, 4096), (3, 128), (5, 144), (33, 2032), (130, 272),
                                 (2, 7168), (257, 64)])
def test_quantize_rows(cl, dtype, r, k):
    x = spread_values(gen(r + k), r, k, dtype)
    check_codes(quantize(cl, x), x.double().numpy(), 1, dtype == torch.bfloat16)


@pytest.mark.parametrize("n,k", [(1, 16), (128, 128), (129, 144), (300, 2032), (64, 4096), (513, 96)])
def test_quantize_blocks(cl, n, k):
    w = spread_values(gen(n + k), n, k, torch.bfloat16)
    c, s = cl.quantize_fp8_blocks(w.cuda(), n, k)
    assert c.dtype == FP8 and c.shape == (n, k)
    check_codes((ref.e4m3(c), s.cpu().numpy()), w.double().numpy(), 128, True)


def test_quantize_halfway_values(cl):
    """bf16 values halfway between two codes for maxima of every mantissa: ties
    to even, whatever 448 / maximum rounds to."""
    rows = []
    for m in range(128, 256):
        top = m * 2.0 ** -7
        mids = (ref.e4m3(np.arange(0, 126, dtype=np.uint8)) +
                ref.e4m3(np.arange(1, 127, dtype=np.uint8))) / 2 * top / 448
        v = torch.from_numpy(np.concatenate([mids, [top, -top]])).to(torch.bfloat16)
        rows.append(v)
    x = torch.stack(rows)
    x[:, 126] = torch.tensor([m * 2.0 ** -7 for m in range(128, 256)]).to(torch.bfloat16)
    q, _ = ref.quotients(x.double().numpy(), 1)
    step = ref.e4m3_step(q)
    assert (np.abs(q / step - np.round(q / step)) == 0.5).sum() > 100  # such ties are there
    check_codes(quantize(cl, x), x.double().numpy(), 1, True)


def test_quantize_infinity_and_nan(cl):
    x = torch.ones(3, 256, dtype=torch.bfloat16)
    x[0, 3] = float("inf")
    x[1, 130] = float("nan")
    c, s = quantize(cl, x)
    v = c * np.repeat(s, 128, 1)
    assert not np.isfinite(v[0, :128]).any() and np.allclose(v[0, 128:], 1, rtol=0.07)
    assert np.isnan(v[1, 130]) and np.isfinite(np.delete(v[1], 130)).all()
    assert np.isfinite(v[2]).all()


def test_quantize_nothing_and_refusals(cl):
    e = torch.empty((0, 32), device="cuda")
    cl.quantize_fp8(e, 0, 32, torch.empty((0, 32), dtype=FP8, device="cuda"),
                    torch.empty((0, 1), device="cuda"))
    x = torch.zeros((4, 32), device="cuda")
    c, s = torch.empty((4, 32), dtype=FP8, device="cuda"), torch.empty((4, 1), device="cuda")
    for a in ((x, 4, 24, c, s), (x.half(), 4, 32, c, s), (x, 4, 32, c.float(), s),
              (x, 4, 32, c, s.double()), (x, 4, 32, c, torch.empty((4, 2), device="cuda")),
              (x, 3, 32, c, s), (x.cpu(), 4, 32, c, s)):
        with pytest.raises(ValueError):
            cl.quantize_fp8(*a)
    flat = torch.zeros(4 * 32 + 1, device="cuda")[1:].view(4, 32)  # rows off 16 bytes
    with pytest.raises(cl.CascadiaInt4Error):
        cl.quantize_fp8(flat, 4, 32, c, s)
    with pytest.raises(ValueError):
        cl.quantize_fp8_blocks(torch.zeros((4, 24), dtype=torch.bfloat16, device="cuda"), 4, 24)
    with pytest.raises(ValueError):
        cl.quantize_fp8_blocks(x, 4, 32)


# ---------------------------------------------------------------------------
# product
# ---------------------------------------------------------------------------

def gemm_case(seed, m, n, k, kind):
    g = gen(seed)
    w, ws = codes(g, n, k), scales(g, ref.blocks(n), ref.blocks(k))
    if kind == "fp8":
        return w, ws, codes(g, m, k), scales(g, m, ref.blocks(k))
    return w, ws, normal(g, m, k, dtype=torch.float32 if kind == "f32" else torch.bfloat16), None


def gemm_ref(w, ws, x, xs):
    """(y, bound) of the product; f32 rows may take a neighbouring code where the
    quotient lies within its rounding of a border."""
    wd, wsd = ref.e4m3(w), ws.double().numpy()
    if xs is not None:
        return ref.gemm(ref.e4m3(x), xs.double().numpy(), wd, wsd)
    q, s = ref.quotients(x.double().numpy(), 1)
    xq = ref.round_e4m3(q)
    y, b = ref.gemm(xq, s, wd, wsd)
    step = ref.e4m3_step(q)
    border = np.abs(np.abs(q - xq) - step / 2) <= 4 * ref.U32 * np.abs(q)
    if x.dtype == torch.bfloat16:  # quotients of bf16 values are exact enough
        border[:] = False
    d = np.where(border, step, 0) * np.repeat(s, 128, 1)[:, :x.shape[1]]
    return y, b + d @ np.abs(wd * ref.spread(wsd, *wd.shape)).T


def eight_bit(w, ws, x, xs):
    n, k = w.shape
    if xs is None:
        q, s = ref.quotients(x.double().numpy(), 1)
        xq = ref.round_e4m3(q)
    else:
        xq, s = ref.e4m3(x), xs.double().numpy()
    return ref.eight_bit_sums(xq * np.repeat(s, 128, 1)[:, :k],
                              ref.e4m3(w) * ref.spread(ws.double().numpy(), n, k))


def check_gemm(cl, w, ws, x, xs, y_dtype, workspace=None):
    m, k = x.shape
    n = w.shape[0]
    y = torch.full((m, n), float("nan"), dtype=y_dtype, device="cuda")
    cl.fp8_gemm(w.cuda(), ws.cuda(), x.cuda(), n, k, m, y,
                x_scales=None if xs is None else xs.cuda(), workspace=workspace)
    want, bound = gemm_ref(w, ws, x, xs)
    if y_dtype == torch.bfloat16:
        if m > 16:  # products of many rows may run on the 8-bit MFMAs
            bound = bound + eight_bit(w, ws, x, xs)
        bound = bound + ref.BF16 * (np.abs(want) + bound)
    off = np.abs(y.double().cpu().numpy() - want) - bound
    assert np.all(off <= 0), (off.max(), np.unravel_index(np.argmax(off), off.shape))
    return y


GEMM_SIZES = [(1, 1, 16), (1, 16, 128), (1, 300, 144), (1, 4096, 2048), (2, 130, 1040),
              (3, 17, 4096), (5, 33, 32), (15, 64, 384), (16, 129, 2064), (17, 256, 128),
              (31, 40, 528), (32, 576, 1024), (33, 15, 272), (48, 128, 640), (63, 31, 160),
              (64, 512, 512), (65, 200, 656), (100, 257, 1152), (128, 128, 128), (129, 385, 400),
              (200, 640, 256), (255, 130, 912), (256, 256, 384), (300, 511, 1296), (513, 144, 528),
              (1000, 48, 80)]


@pytest.mark.parametrize("kind", ["fp8", "bf16", "f32"])
@pytest.mark.parametrize("m,n,k", GEMM_SIZES)
def test_gemm(cl, m, n, k, kind):
    w, ws, x, xs = gemm_case(m + n + k, m, n, k, kind)
    check_gemm(cl, w, ws, x, xs, torch.float32 if (m + n) % 2 else torch.bfloat16)


@pytest.mark.parametrize("m,n,k", [(1, 32, 17408), (2, 40, 33040), (20, 16, 20496), (70, 24, 33040)])
@pytest.mark.parametrize("kind", ["fp8", "bf16"])
def test_gemm_long_rows(cl, m, n, k, kind):
    """More blocks than the few-row kernels hold scales for at once."""
    w, ws, x, xs = gemm_case(m + k, m, n, k, kind)
    check_gemm(cl, w, ws, x, xs, torch.float32)


@pytest.mark.parametrize("m,n,k", [(3500, 3600, 272), (1700, 3600, 400), (1000, 1100, 144),
                                   (4100, 4200, 144), (2300, 8100, 272)])
@pytest.mark.parametrize("y_dtype", [torch.float32, torch.bfloat16])
def test_gemm_many_tiles(cl, m, n, k, y_dtype):
    """Ragged products on the larger tiles: every output written, the rows at the
    tiles' edges and some between against the reference."""
    w, ws, x, xs = gemm_case(m, m, n, k, "fp8")
    y = torch.full((m, n), float("nan"), dtype=y_dtype, device="cuda")
    cl.fp8_gemm(w.cuda(), ws.cuda(), x.cuda(), n, k, m, y, x_scales=xs.cuda())
    assert torch.isfinite(y).all()
    rows = sorted({0, 1, 127, 128, 255, 256, m // 2, m - 2, m - 1, *range(77, m, 997)})
    want, bound = gemm_ref(w, ws, x[rows], xs[rows])
    if y_dtype == torch.bfloat16:
        bound = bound + eight_bit(w, ws, x[rows], xs[rows])
        bound = bound + ref.BF16 * (np.abs(want) + bound)
    assert np.all(np.abs(y[rows].double().cpu().numpy() - want) <= bound)


@pytest.mark.parametrize("y_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m", [1, 4, 20, 70, 300])
def test_gemm_scales_belong_to_their_blocks(cl, m, y_dtype):
    """Scales from 2^-30 to 2^30: a block times another's scale is far off."""
    g = gen(m)
    n, k = 272, 656
    w, ws, x, xs = gemm_case(m, m, n, k, "fp8")
    ws = 2.0 ** torch.randint(-15, 15, ws.shape, generator=g).float()
    xs = 2.0 ** torch.randint(-15, 15, xs.shape, generator=g).float()
    check_gemm(cl, w, ws, x, xs, y_dtype)


@pytest.mark.parametrize("m", [1, 16, 40, 130])
def test_gemm_every_code(cl, m):
    """Every finite code, subnormal ones among them, against exact powers of two."""
    finite = torch.tensor([c for c in range(256) if c & 0x7F != 0x7F], dtype=torch.uint8)
    w = torch.zeros((254, 256), dtype=torch.uint8)
    w[:, :254] = torch.diag(finite)
    x = torch.ones((m, 256)).to(FP8)
    y = torch.empty((m, 254), device="cuda")
    one = torch.ones
    cl.fp8_gemm(w.cuda(), one((2, 2), device="cuda"), x.cuda(), 254, 256, m, y,
                x_scales=one((m, 2), device="cuda"))
    assert np.array_equal(y.double().cpu().numpy(), np.tile(ref.e4m3(finite.numpy()), (m, 1)))


@pytest.mark.parametrize("m,n", [(1, 64), (16, 48), (40, 200), (200, 264)])
def test_gemm_nan_stays_in_its_row(cl, m, n):
    """A NaN code in one token, and one in a weight row, reach their row and
    column only; the codes next to a short last block are not read as values."""
    k = 208
    w, ws, x, xs = gemm_case(1, m, n, k, "fp8")
    xu, wu = x.view(torch.uint8), w.view(torch.uint8)
    xu[m - 1, k - 1] = 0x7F
    wu[n - 3, 0] = 0xFF
    y = torch.empty((m, n), device="cuda")
    cl.fp8_gemm(w.cuda(), ws.cuda(), x.cuda(), n, k, m, y, x_scales=xs.cuda())
    nan = torch.isnan(y).cpu().numpy()
    want = np.zeros((m, n), bool)
    want[m - 1], want[:, n - 3] = True, True
    assert np.array_equal(nan, want)


@pytest.mark.parametrize("m", [1, 9, 33, 150])
def test_gemm_writes_its_rows_only(cl, m):
    n, k = 77, 256
    w, ws, x, xs = gemm_case(2, m, n, k, "fp8")
    buf = torch.full((m * n + 64,), 3.0, device="cuda")
    cl.fp8_gemm(w.cuda(), ws.cuda(), x.cuda(), n, k, m, buf[:m * n], x_scales=xs.cuda())
    assert torch.all(buf[m * n:] == 3.0) and not torch.any(buf[:m * n] == 3.0)


def test_gemm_output_off_its_vector_alignment(cl):
    for m, n in ((1, 64), (20, 64), (150, 256)):
        w, ws, x, xs = gemm_case(m, m, n, 256, "fp8")
        for dt in (torch.float32, torch.bfloat16):
            y = torch.empty(m * n + 1, dtype=dt, device="cuda")[1:]
            z = torch.empty(m * n, dtype=dt, device="cuda")
            for o in (y, z):
                cl.fp8_gemm(w.cuda(), ws.cuda(), x.cuda(), n, 256, m, o, x_scales=xs.cuda())
            assert torch.equal(y, z)


@pytest.mark.parametrize("m,n,k", [(1, 512, 2048), (8, 300, 1040), (70, 256, 4096), (260, 384, 512)])
def test_gemm_is_repeatable(cl, m, n, k):
    w, ws, x, xs = gemm_case(m, m, n, k, "bf16")
    a = [t.cuda() for t in (w, ws, x)]
    ys = [cl.fp8_gemm(*a, n, k, m, torch.empty((m, n), device="cuda")) for _ in range(3)]
    assert torch.equal(ys[0], ys[1]) and torch.equal(ys[0], ys[2])


def test_gemm_refusals(cl):
    w, ws, x, xs = (t.cuda() for t in gemm_case(1, 2, 32, 64, "fp8"))
    y = torch.empty((2, 32), device="cuda")
    xb = torch.zeros((2, 64), dtype=torch.bfloat16, device="cuda")
    ok = dict(x_scales=xs)
    for a, kw in (((w, ws, x, 32, 64, 2, y), {}), ((w, ws, xb, 32, 64, 2, y), ok),
                  ((w, ws, x, 32, 64, 0, y), ok), ((w, ws, x, 32, 72, 2, y), ok),
                  ((w, ws[:, :0], x, 32, 64, 2, y), ok), ((w, ws, x, 31, 64, 2, y), ok),
                  ((w, ws, x, 32, 64, 2, y.half()), ok), ((w, ws, x, 32, 64, 3, y), ok),
                  ((w, ws, xb.half(), 32, 64, 2, y), {}), ((w.cpu(), ws, x, 32, 64, 2, y), ok),
                  ((w, ws.double(), x, 32, 64, 2, y), ok),
                  ((w, ws, x, 32, 64, 2, y), dict(x_scales=xs.view(-1)[:1])),
                  ((w, ws, xb, 32, 64, 2, y),
                   dict(workspace=torch.empty(16, dtype=torch.uint8, device="cuda")))):
        with pytest.raises(ValueError):
            cl.fp8_gemm(*a, **kw)


# ---------------------------------------------------------------------------
# experts
# ---------------------------------------------------------------------------

def moe_case(seed, T, H, I, E, k, x_dtype, ids=None):
    g = gen(seed)
    gu, dn = codes(g, E, 2, I, H), codes(g, E, H, I)
    gus = scales(g, E, 2, ref.blocks(I), ref.blocks(H)) / H ** 0.5
    dns = scales(g, E, ref.blocks(H), ref.blocks(I)) / I ** 0.5
    x = normal(g, T, H, dtype=x_dtype)
    if ids is None:
        ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    w = torch.rand((T, k), generator=g)
    res = normal(g, T, H)
    return gu, gus, dn, dns, x, ids.to(torch.int32), w, res


def moe_ref(case, threshold, residual):
    gu, gus, dn, dns, x, ids, w, _ = case
    out, bound = ref.moe(x.double().numpy(), ref.e4m3(gu), gus.double().numpy(), ref.e4m3(dn),
                         dns.double().numpy(), ids.numpy(), w.double().numpy(), threshold,
                         None if residual is None else residual.double().numpy())
    return out, bound


def run_moe(cl, case, out_dtype, threshold, residual, workspace=None, tiled=True):
    gu, gus, dn, dns, x, ids, w, _ = case
    E, _, I, H = gu.shape
    ex = cl.Fp8Experts(gu.cuda(), gus.cuda(), dn.cuda(), dns.cuda(), E, H, I, tiled=tiled)
    out = torch.full(x.shape, float("nan"), dtype=out_dtype, device="cuda")
    cl.fp8_moe_forward(ex, x.cuda(), out, top_k=ids.shape[1], ids=ids.cuda(), weights=w.cuda(),
                       threshold=threshold, workspace=workspace,
                       residual=None if residual is None else residual.cuda())
    return out


def check_moe(cl, case, out_dtype=torch.bfloat16, threshold=0.0, residual=True):
    res = case[-1].to(out_dtype) if residual else None
    out = run_moe(cl, case, out_dtype, threshold, res).double().cpu().numpy()
    want, bound = moe_ref(case, threshold, res)
    if out_dtype == torch.bfloat16:
        bound = bound + ref.BF16 * (np.abs(want) + bound)
    off = np.abs(out - want) - bound
    assert np.all(off <= 0), (off.max(), np.unravel_index(np.argmax(off), off.shape))
    # as a whole: bf16 slots and output, 2 x 2^-9; 8-bit sums of up to 5e-5 move at
    # most 2 sqrt(2) 5e-5 / 2^-4 of the codes by a step of 2^-3 of them: 6e-3
    assert np.linalg.norm(out - want) <= 1e-2 * np.linalg.norm(want)


@pytest.mark.parametrize("T,H,I,E,k", [
    (1, 256, 128, 8, 2), (1, 16, 16, 1, 1), (1, 1040, 400, 16, 8), (2, 144, 272, 4, 4),
    (3, 512, 96, 5, 3), (17, 256, 256, 3, 2), (40, 128, 144, 2, 1), (33, 272, 128, 64, 16),
    (1, 64, 144, 20, 16), (1, 32, 4096, 16, 16), (120, 16, 16, 700, 8), (200, 32, 16, 700, 8),
    (70, 256, 160, 2, 2), (150, 144, 128, 3, 2), (400, 128, 272, 5, 4), (600, 64, 48, 3, 2)])
@pytest.mark.parametrize("x_dtype", [torch.float32, torch.bfloat16])
def test_moe(cl, T, H, I, E, k, x_dtype):
    case = moe_case(T + H + I, T, H, I, E, k, x_dtype)
    check_moe(cl, case, torch.float32 if (T + k) % 2 else torch.bfloat16, residual=T % 3 != 0)


@pytest.mark.parametrize("T,H,I,E,k", [(8, 256, 144, 1, 1), (16, 400, 272, 4, 2),
                                       (15, 144, 128, 4, 2), (2, 64, 1040, 1, 16)])
def test_moe_about_eight_rows_per_expert(cl, T, H, I, E, k):
    """Either side of the step from 16-row chunks to tiles, and a few tokens on tiles."""
    ids = torch.randint(0, E, (T, k), generator=gen(T), dtype=torch.int32)
    check_moe(cl, moe_case(T + H, T, H, I, E, k, torch.bfloat16, ids))


@pytest.mark.parametrize("T,H,I,E,k", [(1, 400, 272, 5, 3), (9, 144, 1040, 4, 2),
                                       (90, 272, 400, 3, 2), (300, 128, 16, 2, 1)])
def test_moe_tiled_codes_are_the_same_codes(cl, T, H, I, E, k):
    case = moe_case(T, T, H, I, E, k, torch.bfloat16)
    a, b = (run_moe(cl, case, torch.float32, 0.0, None, tiled=t) for t in (True, False))
    assert torch.equal(a, b)


@pytest.mark.parametrize("count,n,k", [(1, 1, 16), (3, 128, 128), (2, 130, 272), (5, 300, 144)])
def test_tile_weights(cl, count, n, k):
    w = codes(gen(n), count, n, k).view(torch.uint8).cuda()
    L = cl.lib()
    per = L.cascadia_int4_fp8_tiled_bytes(n, k)
    nb, kb = ref.blocks(n), ref.blocks(k)
    assert per == nb * kb * 128 * 128
    out = torch.full((count * per + 64,), 7, dtype=torch.uint8, device="cuda")
    cl.check("tile", L.cascadia_int4_fp8_tile_weights(count, n, k, w.data_ptr(), out.data_ptr(),
                                                      torch.cuda.current_stream().cuda_stream))
    want = torch.zeros((count, nb * 128, kb * 128), dtype=torch.uint8)
    want[:, :n, :k] = w.cpu()
    want = want.view(count, nb, 128, kb, 128).permute(0, 1, 3, 2, 4).reshape(-1)
    assert torch.equal(out[:-64].cpu(), want) and torch.all(out[-64:] == 7)


def test_moe_one_expert_takes_every_token(cl):
    ids = torch.zeros((140, 2), dtype=torch.int32)
    ids[:, 1] = 3
    check_moe(cl, moe_case(1, 140, 128, 144, 4, 2, torch.bfloat16, ids))


def test_moe_slots_left_out(cl):
    """Padding ids, ids past the layer, weights below the threshold, a token with
    no slot at all, the same expert twice in one token."""
    g = gen(9)
    ids = torch.randint(0, 6, (40, 3), generator=g)
    ids[4] = -1
    ids[5, 0], ids[6, 1], ids[7, 2] = 6, 2 ** 31 - 1, -2 ** 31
    ids[8] = 2
    case = moe_case(2, 40, 160, 256, 6, 3, torch.bfloat16, ids)
    w = case[6]
    w[10], w[11, 1] = 0.05, 0.0999
    check_moe(cl, case, threshold=0.1)
    check_moe(cl, case, torch.float32, threshold=0.1, residual=False)
    # rows of tokens without slots are the residual
    out = run_moe(cl, case, torch.bfloat16, 0.1, case[-1].to(torch.bfloat16))
    assert torch.equal(out[[4, 10]].cpu(), case[-1].to(torch.bfloat16)[[4, 10]])


def test_moe_every_slot_left_out(cl):
    ids = torch.full((3, 2), -1)
    case = moe_case(3, 3, 128, 128, 4, 2, torch.float32, ids)
    assert torch.all(run_moe(cl, case, torch.float32, 0.0, None) == 0)


@pytest.mark.parametrize("T", [1, 20, 150])
def test_moe_nan_stays_in_its_token(cl, T):
    case = moe_case(4, T, 128, 128, 4, 2, torch.float32)
    case[4][T // 2, 7] = float("nan")
    out = run_moe(cl, case, torch.float32, 0.0, None).cpu()
    bad = torch.isnan(out).any(1)
    assert bad[T // 2] and int(bad.sum()) == 1


@pytest.mark.parametrize("T", [1, 20, 200])
def test_moe_in_place(cl, T):
    """out is the residual, or x itself."""
    case = moe_case(7, T, 144, 128, 4, 2, torch.bfloat16)
    gu, gus, dn, dns, x, ids, w, res = (t.cuda() for t in case)
    ex = cl.Fp8Experts(gu, gus, dn, dns, 4, 144, 128)
    kw = dict(top_k=2, ids=ids, weights=w)
    res = res.to(torch.bfloat16)
    want = cl.fp8_moe_forward(ex, x, torch.empty_like(x), residual=res, **kw)
    a = res.clone()
    assert torch.equal(cl.fp8_moe_forward(ex, x, a, residual=a, **kw), want)
    want = cl.fp8_moe_forward(ex, x, torch.empty_like(x), residual=x, **kw)
    b = x.clone()
    assert torch.equal(cl.fp8_moe_forward(ex, b, b, residual=b, **kw), want)


def test_one_workspace_serves_smaller_calls(cl):
    """A workspace of the largest batch, for every smaller one."""
    n, k = 320, 1040
    w, ws, x, xs = (t.cuda() for t in gemm_case(8, 400, n, k, "fp8"))
    for kind, scales_of in ((x, xs), (x.float(), None)):
        buf = torch.empty(cl.fp8_gemm_workspace_bytes(n, k, 400, kind.dtype), dtype=torch.uint8,
                          device="cuda")
        for m in (400, 300, 129, 65, 64, 33, 17, 2, 1):
            sc = None if scales_of is None else scales_of[:m]
            a, b = (torch.empty((m, n), device="cuda") for _ in range(2))
            cl.fp8_gemm(w, ws, kind[:m], n, k, m, a, x_scales=sc, workspace=buf)
            cl.fp8_gemm(w, ws, kind[:m], n, k, m, b, x_scales=sc)
            assert torch.equal(a, b)
    gu, gus, dn, dns, x, ids, wt, _ = (t.cuda() for t in moe_case(8, 200, 144, 400, 6, 2, torch.float32))
    ex = cl.Fp8Experts(gu, gus, dn, dns, 6, 144, 400)
    buf = torch.empty(cl.fp8_moe_workspace_bytes(ex, 2, 200), dtype=torch.uint8, device="cuda")
    for t in (200, 100, 48, 47, 20, 2, 1):
        a, b = (torch.empty((t, 144), device="cuda") for _ in range(2))
        kw = dict(top_k=2, ids=ids[:t], weights=wt[:t])
        cl.fp8_moe_forward(ex, x[:t], a, workspace=buf, **kw)
        cl.fp8_moe_forward(ex, x[:t], b, **kw)
        assert torch.equal(a, b)


@pytest.mark.parametrize("T", [1, 30, 200])
def test_moe_is_repeatable(cl, T):
    case = moe_case(5, T, 256, 272, 7, 3, torch.bfloat16)
    a = [run_moe(cl, case, torch.float32, 0.0, None) for _ in range(3)]
    assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2])


def test_moe_refusals(cl):
    gu, gus, dn, dns, x, ids, w, _ = (t.cuda() for t in moe_case(6, 2, 64, 32, 3, 2, torch.float32))
    for a in ((gu, gus, dn, dns, 2, 64, 32), (gu, gus, dn, dns, 3, 64, 48),
              (gu, gus[:, :1].contiguous(), dn, dns, 3, 64, 32), (gu.cpu(), gus, dn, dns, 3, 64, 32),
              (gu, gus, dn.float(), dns, 3, 64, 32), (gu, gus, dn, dns, 0, 64, 32)):
        with pytest.raises(ValueError):
            cl.Fp8Experts(*a)
    ex = cl.Fp8Experts(gu, gus, dn, dns, 3, 64, 32)
    out = torch.empty_like(x)
    ok = dict(top_k=2, ids=ids, weights=w)
    small = torch.empty(64, dtype=torch.uint8, device="cuda")
    for a, kw in (((x, out), {**ok, "top_k": 3}), ((x, out), {**ok, "ids": ids.long()}),
                  ((x, out), {**ok, "weights": w[:1]}), ((x.half(), out), ok),
                  ((x, out.to(torch.float16)), ok), ((x[:0], out[:0]), ok),
                  ((x, out), {**ok, "residual": out.to(torch.bfloat16)}),
                  ((x, out), {**ok, "workspace": small}), ((x, out), {**ok, "ids": ids.cpu()}),
                  ((x, out), {**ok, "top_k": 0})):
        with pytest.raises(ValueError):
            cl.fp8_moe_forward(ex, *a, **kw)


# ---------------------------------------------------------------------------
# as they are used together
# ---------------------------------------------------------------------------

def layer_case(T, seed=11):
    g = gen(seed)
    H, I, E, k = 256, 144, 24, 4
    gate, bias = normal(g, E, H, dtype=torch.bfloat16), normal(g, E) * 0.05
    w1, w2 = normal(g, E, 2, I, H, dtype=torch.bfloat16), normal(g, E, H, I, dtype=torch.bfloat16)
    return H, I, E, k, gate, bias, w1 / H ** 0.5, w2 / I ** 0.5, normal(g, T, H, dtype=torch.bfloat16)


def load_layer(cl, H, I, E, w1, w2):
    """A layer's bf16 experts quantised as they are loaded."""
    gu = torch.empty((E, 2, I, H), dtype=FP8, device="cuda")
    gus = torch.empty((E, 2, ref.blocks(I), ref.blocks(H)), device="cuda")
    dn = torch.empty((E, H, I), dtype=FP8, device="cuda")
    dns = torch.empty((E, ref.blocks(H), ref.blocks(I)), device="cuda")
    for e in range(E):
        for j in (0, 1):
            gu[e, j], gus[e, j] = cl.quantize_fp8_blocks(w1[e, j].cuda(), I, H)
        dn[e], dns[e] = cl.quantize_fp8_blocks(w2[e].cuda(), H, I)
    return (gu, gus, dn, dns), cl.Fp8Experts(gu, gus, dn, dns, E, H, I)


class Layer:
    """Router product, choice and experts of a layer over its own buffers."""

    def __init__(self, cl, T, seed=11):
        self.cl, self.T = cl, T
        (self.H, self.I, self.E, self.k, gate, self.bias, w1, w2, x) = layer_case(T, seed)
        self.x = x.cuda()
        self.gate, self.gate_s = cl.quantize_fp8_blocks(gate.cuda(), self.E, self.H)
        self.given, self.ex = load_layer(cl, self.H, self.I, self.E, w1, w2)
        self.bias = self.bias.cuda()
        self.logits = torch.empty((T, self.E), device="cuda")
        self.ids = torch.empty((T, self.k), dtype=torch.int32, device="cuda")
        self.w = torch.empty((T, self.k), device="cuda")
        self.out = torch.empty_like(self.x)
        need = max(256, cl.fp8_gemm_workspace_bytes(self.E, self.H, T, self.x.dtype))
        self.ws1 = torch.empty(need, dtype=torch.uint8, device="cuda")
        self.ws2 = torch.empty(cl.fp8_moe_workspace_bytes(self.ex, self.k, T), dtype=torch.uint8,
                               device="cuda")

    def run(self, own_workspace=True):
        cl = self.cl
        a, b = (self.ws1, self.ws2) if own_workspace else (None, None)
        cl.fp8_gemm(self.gate, self.gate_s, self.x, self.E, self.H, self.T, self.logits,
                    workspace=a)
        cl.route_experts(self.logits, self.k, self.ids, self.w, bias=self.bias, n_groups=4,
                         top_groups=2, scale=2.5)
        cl.fp8_moe_forward(self.ex, self.x, self.out, top_k=self.k, ids=self.ids, weights=self.w,
                           residual=self.x, workspace=b)
        return self.out


@pytest.mark.parametrize("T", [1, 6, 40, 170])
def test_layer_from_router_to_experts(cl, T):
    L = Layer(cl, T)
    out = L.run().double().cpu().numpy()
    # each step against the reference of what it was given
    y, b = gemm_ref(L.gate.cpu(), L.gate_s.cpu(), L.x.cpu(), None)
    assert np.all(np.abs(L.logits.double().cpu().numpy() - y) <= b)
    ids, w = ref.route(L.logits.double().cpu().numpy(), L.k, "sigmoid",
                       L.bias.double().cpu().numpy(), 4, 2, 2, True, 2.5)
    assert np.array_equal(L.ids.cpu().numpy(), ids)
    gu, gus, dn, dns = L.given
    want, bound = ref.moe(L.x.double().cpu().numpy(), ref.e4m3(gu), gus.double().cpu().numpy(),
                          ref.e4m3(dn), dns.double().cpu().numpy(), ids,
                          L.w.double().cpu().numpy(), 0.0, L.x.double().cpu().numpy())
    bound = bound + ref.BF16 * (np.abs(want) + bound)
    assert np.all(np.abs(out - want) <= bound)


@pytest.mark.parametrize("T", [1, 12, 140])
def test_layer_in_a_graph(cl, T):
    """Recorded once and replayed on new inputs between eager calls."""
    L, other = Layer(cl, T), Layer(cl, T, seed=12)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        L.run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        L.run()
    for step in range(4):
        L.x.copy_(normal(gen(step), T, L.H, dtype=torch.bfloat16))
        L.out.zero_(), L.ids.zero_(), L.logits.zero_()
        graph.replay()
        other.run(own_workspace=False)
        torch.cuda.synchronize()
        got = [t.clone() for t in (L.out, L.ids, L.w, L.logits)]
        L.run()
        assert all(torch.equal(a, b) for a, b in zip(got, (L.out, L.ids, L.w, L.logits)))


def test_layer_in_a_graph_over_the_librarys_workspace(cl):
    T = 20
    L = Layer(cl, T)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = L.run(own_workspace=False).clone()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        L.run(own_workspace=False)
    other = Layer(cl, 3 * T, seed=5)
    for _ in range(3):
        L.out.zero_()
        graph.replay()
        other.run(own_workspace=False)
        torch.cuda.synchronize()
        assert torch.equal(L.out, want)


def test_layers_on_two_streams(cl):
    """Calls without a workspace on two streams at once."""
    layers = [Layer(cl, 60, seed=s) for s in (21, 22)]
    want = [L.run(own_workspace=False).clone() for L in layers]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    for L in layers:
        L.out.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for L, s in zip(layers, streams):
            with torch.cuda.stream(s):
                L.run(own_workspace=False)
    torch.cuda.synchronize()
    assert all(torch.equal(L.out, w) for L, w in zip(layers, want))


def test_int4_layer_takes_the_chosen_experts(cl, orc):
    """route_experts feeds the INT4 layer's ROUTE_IDS form."""
    g = gen(31)
    E, H, I, k, T = 12, 256, 128, 3, 9
    per = cl.expert_bytes(H, I, 32)
    stride = (per + 255) // 256 * 256
    blobs = torch.randint(0, 256, (stride * E,), dtype=torch.uint8, generator=g).cuda()
    view = blobs.view(E, stride)
    at = 0
    for rows, cols in ((I, H), (I, H), (H, I)):
        at += rows * cols // 2
        n = rows * cols // 32
        view[:, at:at + 2 * n] = (torch.rand((E, n), generator=g) * 0.02).to(torch.bfloat16).view(
            torch.uint8).cuda()
        at += 2 * n
    ex = cl.MoEExperts.from_crate(blobs, E, H, I, 32, cl.SCALE_BF16, stride)
    x, logits, bias = normal(g, T, H).cuda(), normal(g, T, E).cuda(), (normal(g, E) * 0.1).cuda()
    ids = torch.empty((T, k), dtype=torch.int32, device="cuda")
    w = torch.empty((T, k), device="cuda")
    cl.route_experts(logits, k, ids, w, bias=bias, scale=2.0)
    a, b = torch.empty_like(x), torch.empty_like(x)
    ids2 = torch.empty_like(ids)
    cl.moe_forward(ex, x, a, top_k=k, ids=ids, weights=w, mode=cl.ROUTE_IDS)
    cl.moe_forward(ex, x, b, top_k=k, logits=logits, bias=bias, scale=2.0, ids_out=ids2)
    assert torch.equal(ids, ids2)
    # the same ids; weights within a few roundings of each other
    assert torch.allclose(a, b, rtol=0, atol=float(b.abs().max()) * 32 * 2.0 ** -24)
