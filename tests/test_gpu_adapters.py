"""Low-rank adapters of many requests on the GPU against the 64-bit reference
(tokens_ref), with bounds that count the roundings."""
import numpy as np
import pytest
import torch

import tokens_ref as ref

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
NAN = float("nan")


@pytest.fixture(scope="module")
def cl():
    import cascadia_amd

    return cascadia_amd


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def plan(cl, ids, E):
    T = ids.numel()
    off, slots, rows = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (E + 1, T, T))
    cl.sort_tokens(ids.cuda(), 1, E, off, slots, rows)
    return off, slots


def case(seed, T, E, R, K, N, x_type, base_type, mixed=True, bare=0.25):
    """a, b (NaN past an adapter's rank), ranks, scales, ids, x (NaN in rows without an
    adapter), base."""
    g = gen(seed)
    a = (torch.randn((E, R, K), generator=g) / K ** 0.5).to(BF16)
    b = (torch.randn((E, N, R), generator=g) / R ** 0.5).to(BF16)
    ranks = torch.randint(0, R + 1, (E,), generator=g, dtype=torch.int32) if mixed else torch.full(
        (E,), R, dtype=torch.int32)
    for i, r in enumerate(ranks.tolist()):
        a[i, r:] = NAN
        b[i, :, r:] = NAN
    scales = torch.rand(E, generator=g) * 3 - 1
    ids = torch.randint(0, E, (T,), generator=g, dtype=torch.int32)
    wild = torch.tensor([-1, E, -2 ** 31, 2 ** 31 - 1])[torch.randint(0, 4, (T,), generator=g)].int()
    ids = torch.where(torch.rand(T, generator=g) < bare, wild, ids)
    x = torch.randn((T, K), generator=g).to(x_type)
    x[(ids < 0) | (ids >= E)] = NAN
    base = None if base_type is None else torch.randn((T, N), generator=g).to(base_type)
    return a, b, ranks, scales, ids, x, base


def host(t):
    return None if t is None else t.double().cpu().numpy()


def check(cl, c, y_type, workspace=True):
    a, b, ranks, scales, ids, x, base = c
    E, R, _ = a.shape
    T, N = len(ids), b.shape[1]
    off, slots = plan(cl, ids, E)
    A = cl.Adapters(a.cuda(), b.cuda(), ranks=ranks.cuda(), scales=scales.cuda())
    ws = None
    if workspace:
        ws = torch.full((cl.adapters_workspace_bytes(A, T),), 255, dtype=torch.uint8, device="cuda")
    ys = torch.full((T + 1, N), 77.0, dtype=y_type, device="cuda")
    cl.adapters_forward(A, x.cuda(), off, slots, ys[:T], workspace=ws,
                        base=None if base is None else base.cuda())
    want, bound = ref.adapters(host(a), host(b), ranks.tolist(), scales.tolist(), ids.tolist(), host(x),
                               host(base), y_type is BF16)
    got = host(ys)
    assert np.all(got[T] == 77.0)  # the row behind
    bad = ~(np.abs(got[:T] - want) <= bound)
    assert not bad.any(), (np.argwhere(bad)[:4], got[:T][bad][:4], want[bad][:4], bound[bad][:4])
    return ys[:T]


SHAPES = [  # T, E, R, K, N
    (1, 1, 8, 8, 1), (1, 3, 16, 128, 64), (2, 5, 24, 136, 17), (15, 4, 16, 1000, 255),
    (16, 1, 32, 256, 256), (17, 9, 40, 520, 65), (64, 64, 8, 264, 300), (65, 2, 64, 512, 129),
    (130, 1, 72, 200, 67), (300, 7, 128, 392, 47), (33, 1024, 8, 72, 40), (40, 3, 256, 136, 80),
    (129, 130, 16, 640, 1000)]


@pytest.mark.parametrize("T,E,R,K,N", SHAPES)
@pytest.mark.parametrize("x_type,base_type,y_type", [
    (BF16, BF16, BF16), (F32, F32, F32), (BF16, F32, BF16), (F32, BF16, F32), (BF16, None, F32),
    (F32, None, BF16)])
def test_matches_the_definition(cl, T, E, R, K, N, x_type, base_type, y_type):
    check(cl, case(T + R, T, E, R, K, N, x_type, base_type), y_type)


@pytest.mark.parametrize("T,E,R,K,N", [(1, 16, 16, 4096, 4096), (64, 100, 64, 4096, 2050),
                                       (3, 4, 16, 14336, 512), (257, 6, 32, 7168, 384)])
@pytest.mark.parametrize("x_type,y_type", [(BF16, BF16), (F32, F32)])
def test_long_rows(cl, T, E, R, K, N, x_type, y_type):
    check(cl, case(T + K, T, E, R, K, N, x_type, x_type, bare=0.1), y_type, workspace=False)


@pytest.mark.parametrize("y_type", [BF16, F32])
def test_rank_zero_and_no_adapter_at_all(cl, y_type):
    c = list(case(3, 70, 5, 16, 136, 100, BF16, y_type, bare=0.0))
    c[2] = torch.zeros(5, dtype=torch.int32)
    c[0][:], c[1][:] = NAN, NAN
    y = check(cl, c, y_type)
    assert torch.equal(y.cpu(), c[6])  # base itself
    c = list(case(4, 70, 5, 16, 136, 100, BF16, y_type, bare=1.0))
    y = check(cl, c, y_type)
    assert torch.equal(y.cpu(), c[6])
    c[6] = None
    assert not check(cl, c, y_type).any()


def test_ranks_past_the_limits_are_clamped(cl):
    c = list(case(5, 20, 3, 16, 64, 40, BF16, BF16, mixed=False))
    a, b, _, scales, ids, x, base = c
    off, slots = plan(cl, ids, 3)
    ys = []
    for r in ([16, 16, 0], [17, 2 ** 31 - 1, -5]):
        A = cl.Adapters(a.cuda(), b.cuda(), ranks=torch.tensor(r, dtype=torch.int32).cuda(),
                        scales=scales.cuda())
        ys.append(cl.adapters_forward(A, x.cuda(), off, slots, torch.empty_like(base.cuda()),
                                      base=base.cuda()))
    assert torch.equal(*ys)


def test_without_ranks_and_scales(cl):
    c = case(6, 40, 3, 24, 72, 50, F32, F32, mixed=False)
    a, b, _, _, ids, x, base = c
    off, slots = plan(cl, ids, 3)
    A = cl.Adapters(a.cuda(), b.cuda())
    y = cl.adapters_forward(A, x.cuda(), off, slots, torch.empty_like(base.cuda()), base=base.cuda())
    want, bound = ref.adapters(host(a), host(b), [24] * 3, [1.0] * 3, ids.tolist(), host(x), host(base),
                               False)
    assert np.all(np.abs(host(y) - want) <= bound)


@pytest.mark.parametrize("t", [BF16, F32])
def test_in_place_and_strides(cl, t):
    """Parts of wider buffers at odd places; ys over base; what lies beside stays."""
    T, K, N = 90, 136, 77
    a, b, ranks, scales, ids, x, base = case(7, T, 6, 16, K, N, t, t)
    off, slots = plan(cl, ids, 6)
    A = cl.Adapters(a.cuda(), b.cuda(), ranks=ranks.cuda(), scales=scales.cuda())
    y0 = cl.adapters_forward(A, x.cuda(), off, slots, torch.empty((T, N), dtype=t, device="cuda"),
                             base=base.cuda())
    wide_x = torch.full((T, K + 9), NAN, dtype=t, device="cuda")
    wide_x[:, 3:3 + K] = x
    wide = torch.full((T, N + 31), 5.0, dtype=t, device="cuda")
    wide[:, 13:13 + N] = base
    part = wide[:, 13:13 + N]
    cl.adapters_forward(A, wide_x[:, 3:3 + K], off, slots, part, base=part)
    assert torch.equal(part, y0)
    assert bool((wide[:, :13] == 5).all()) and bool((wide[:, 13 + N:] == 5).all())
    other = torch.full((T, 2 * N), 5.0, dtype=t, device="cuda")
    wide[:, 13:13 + N] = base
    cl.adapters_forward(A, wide_x[:, 3:3 + K], off, slots, other[:, N - 8:2 * N - 8], base=part)
    assert torch.equal(other[:, N - 8:2 * N - 8], y0) and bool((other[:, :N - 8] == 5).all())


@pytest.mark.parametrize("x_type,y_type", [(BF16, BF16), (F32, F32)])
def test_infinities_and_nan_stay_in_their_rows(cl, x_type, y_type):
    T, E, R, K, N = 35, 2, 16, 136, 70
    a, b, ranks, scales, ids, x, base = case(8, T, E, R, K, N, x_type, y_type, mixed=False, bare=0.0)
    clean = check(cl, (a, b, ranks, scales, ids, x, base), y_type)
    x = x.clone()
    x[4, 7], x[9, 100] = NAN, float("inf")
    base = base.clone()
    base[20, 3], base[21, 5] = float("inf"), NAN
    off, slots = plan(cl, ids, E)
    A = cl.Adapters(a.cuda(), b.cuda(), scales=scales.cuda())
    y = cl.adapters_forward(A, x.cuda(), off, slots, torch.empty_like(clean), base=base.cuda())
    keep = torch.ones((T, N), dtype=torch.bool, device="cuda")
    keep[4], keep[9], keep[20, 3], keep[21, 5] = False, False, False, False
    assert torch.equal(y[keep], clean[keep])
    assert bool(y[4].isnan().all()) and bool((~y[9].isfinite()).all())
    assert y[20, 3] == float("inf") and bool(y[21, 5].isnan())
    # an inner value that is infinite alone: infinities, no NaN
    x1 = torch.zeros((1, K), dtype=x_type)
    x1[0, 0] = float("inf")
    a1, b1 = torch.zeros((1, 8, K), dtype=BF16), torch.ones((1, N, 8), dtype=BF16)
    a1[0, :, 0] = 1.0
    off, slots = plan(cl, torch.zeros(1, dtype=torch.int32), 1)
    y = cl.adapters_forward(cl.Adapters(a1.cuda(), b1.cuda()), x1.cuda(), off, slots,
                            torch.empty((1, N), dtype=y_type, device="cuda"))
    # (0 * inf of the other columns: NaN in the inner product itself where K > 1)
    assert bool((~y.isfinite()).all())


def test_wrong_plans_stay_within_the_buffers(cl):
    """Offsets and slots that sort_tokens never gives: rows outside are left out."""
    a, b, ranks, scales, ids, x, base = case(10, 20, 3, 16, 64, 40, BF16, BF16, bare=0.0)
    A = cl.Adapters(a.cuda(), b.cuda(), ranks=ranks.cuda(), scales=scales.cuda())
    for off in ([0, 50, -3, 20], [-5, 2 ** 31 - 1, -2 ** 31, 7], [9, 9, 9, 9]):
        for slots in (torch.arange(20) - 5, torch.full((20,), 2 ** 31 - 1)):
            buf = torch.full((24, 40), 3.0, dtype=BF16, device="cuda")
            cl.adapters_forward(A, x.cuda(), torch.tensor(off, dtype=torch.int32).cuda(),
                                slots.int().cuda(), buf[2:22], base=base.cuda())
            assert bool((buf[:2] == 3).all()) and bool((buf[22:] == 3).all())


def test_no_rows_and_refusals(cl):
    T, K, N, E = 6, 64, 40, 3
    a, b, ranks, scales, ids, x, base = case(11, T, E, 16, K, N, BF16, BF16)
    A = cl.Adapters(a.cuda(), b.cuda(), ranks=ranks.cuda(), scales=scales.cuda())
    off, slots = plan(cl, ids, E)
    e = torch.empty((0, K), dtype=BF16, device="cuda")
    cl.adapters_forward(A, e, off, slots[:0], torch.empty((0, N), dtype=BF16, device="cuda"))
    x, base, y = x.cuda(), base.cuda(), torch.empty((T, N), dtype=BF16, device="cuda")
    for bad in (dict(offsets=off[:3]), dict(slots=slots.long()), dict(xs=x[:5]), dict(xs=x[:, :56]),
                dict(xs=x.half()), dict(xs=x.t()), dict(ys=y[:, :39]), dict(ys=y.double()),
                dict(base=base[:5]), dict(base=y.view(torch.int16)), dict(xs=x.cpu()),
                dict(ys=torch.empty((N, T), dtype=BF16, device="cuda").t()),
                dict(ys=y[:1].expand(T, N)),
                dict(workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))):
        args = dict(adapters=A, xs=x, offsets=off, slots=slots, ys=y, base=base)
        args.update(bad)
        with pytest.raises(ValueError):
            cl.adapters_forward(**args)
    wide = torch.empty((T, 2 * N), dtype=BF16, device="cuda")
    with pytest.raises(ValueError):  # in place, another stride
        cl.adapters_forward(A, x, off, slots, wide[:, :N], base=wide.view(-1)[:T * N].view(T, N))
    for bad in ((a[:, :12], b[:, :, :12]), (a[:2], b), (a, b[:, :, :8]), (a.float(), b), (a[0], b[0]),
                (a[:, :, :60], b)):
        with pytest.raises(ValueError):
            cl.Adapters(*(t.contiguous().cuda() for t in bad))
    with pytest.raises(ValueError):
        cl.Adapters(a.cuda(), b.cuda(), ranks=ranks[:2].cuda())
    with pytest.raises(ValueError):
        cl.Adapters(a.cuda(), b.cuda(), scales=scales.double().cuda())


def test_repeats_streams_and_recorded_calls(cl):
    """The same bits from every run, stream and replay; ranks and scales as of the call."""
    T, E, R, K, N = 200, 12, 32, 1040, 600
    a, b, ranks, scales, ids, x, base = (t.cuda() for t in case(12, T, E, R, K, N, F32, F32,
                                                                mixed=False))
    A = cl.Adapters(a, b, ranks=ranks, scales=scales)
    ws = torch.empty(cl.adapters_workspace_bytes(A, T), dtype=torch.uint8, device="cuda")
    off, slots, rows = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (E + 1, T, T))
    y = torch.empty((T, N), device="cuda")

    def call(out, own=True):
        cl.sort_tokens(ids, 1, E, off, slots, rows)
        cl.adapters_forward(A, x, off, slots, out, base=base, workspace=ws if own else None)
        return out

    other = torch.flip(ids, (0,)).clone()
    bad = ~((ids >= 0) & (ids < E))
    x[bad] = 1.0
    want = []
    keep = ids.clone()
    for i in (keep, other):
        ids.copy_(i)
        want.append(call(torch.empty_like(y)).clone())
    assert torch.equal(want[1], call(torch.empty_like(y), own=False))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = call(torch.empty_like(y))
    s.synchronize()
    assert torch.equal(z, want[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(y)
    for i in (0, 1, 0, 0):
        ids.copy_((keep, other)[i])
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i])
        call(torch.empty_like(y))
    scales.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, base)


@pytest.mark.parametrize("rows", [1, 40])
def test_unit_weights_return_x(cl, rows):
    """Adapters that pick columns: f32 values come back whole, from the largest to small
    ones.  (A value's three planes are added twice, in the inner product and in the
    outer one: two additions each, of 2^-23 at most.)"""
    K, N, R = 264, 96, 24
    g = gen(13)
    cols = torch.randperm(K, generator=g)[:R]
    a, b = torch.zeros((1, R, K), dtype=BF16), torch.zeros((1, N, R), dtype=BF16)
    a[0, torch.arange(R), cols] = 1.0
    b[0, torch.arange(N), torch.arange(N) % R] = 1.0
    for scale in (1.0, 3.4e38, 1e-30):
        x = (torch.rand((rows, K), generator=g) * 2 - 1) * scale
        x[0, cols[0]] = scale
        off, slots = plan(cl, torch.zeros(rows, dtype=torch.int32), 1)
        y = cl.adapters_forward(cl.Adapters(a.cuda(), b.cuda()), x.cuda(), off, slots,
                                torch.empty((rows, N), device="cuda"))
        want = host(x[:, cols])[:, np.arange(N) % R]
        assert np.all(np.abs(host(y) - want) <= 2.0 ** -21 * np.abs(want))


def test_signs_of_zero_rows_and_small_values(cl):
    """Rows without an adapter: base as it is, subnormal values among it."""
    T, E, N, K = 40, 2, 100, 16
    base = torch.tensor([1e-40, -3e-39, 1.4e-45, 0.0, 1.1754944e-38]).repeat(T, N // 5)
    off, slots = plan(cl, torch.full((T,), -1, dtype=torch.int32), E)
    A = cl.Adapters(torch.ones((E, 8, K), dtype=BF16, device="cuda"),
                    torch.ones((E, N, 8), dtype=BF16, device="cuda"))
    x = torch.ones((T, K), device="cuda")
    for b in (base, base.to(BF16)):
        for t in (F32, BF16):
            y = cl.adapters_forward(A, x, off, slots, torch.empty((T, N), dtype=t, device="cuda"),
                                    base=b.cuda())
            assert torch.equal(y.cpu(), b.to(t))
