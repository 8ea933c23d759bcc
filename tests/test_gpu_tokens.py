"""Tokens sorted by expert and back on the GPU, each against the 64-bit reference
(tokens_ref) with bounds that count its roundings."""
import numpy as np
import pytest
import torch

import tokens_ref as ref

pytestmark = pytest.mark.gpu
F32, BF16, FP8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
NAN = float("nan")


@pytest.fixture(scope="module")
def cl():
    import cascadia_amd

    return cascadia_amd


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def some_ids(g, T, k, E, padded=0, wild=0.1):
    """Distinct experts per token where there are enough; some slots with no expert."""
    if k <= E:
        ids = torch.rand((T, E), generator=g).topk(k, dim=1).indices.int()
    else:
        ids = torch.randint(0, E, (T, k), generator=g, dtype=torch.int32)
    bad = torch.tensor([-1, -7, E, E + 3, 2 ** 31 - 1, -2 ** 31])
    ids = torch.where(torch.rand((T, k), generator=g) < wild,
                      bad[torch.randint(0, 6, (T, k), generator=g)].int(), ids)
    if padded:
        ids[-padded:] = -1
    return ids


def run_sort(cl, ids, E, weights=None, threshold=0.0, workspace=None):
    T, k = ids.shape
    buf = torch.full((E + 1 + 2 * T * k + 3,), -99, dtype=torch.int32, device="cuda")
    off, slots, rows = buf[:E + 1], buf[E + 2:E + 2 + T * k], buf[E + 3 + T * k:E + 3 + 2 * T * k]
    cl.sort_tokens(ids.cuda(), k, E, off, slots, rows, threshold=threshold, workspace=workspace,
                   weights=None if weights is None else weights.cuda())
    assert buf[E + 1] == -99 and buf[E + 2 + T * k] == -99
    return off.cpu().numpy(), slots.cpu().numpy(), rows.view(T, k).cpu().numpy()


def check_sort(cl, ids, E, weights=None, threshold=0.0):
    got = run_sort(cl, ids, E, weights, threshold)
    want = ref.sort(ids.numpy(), E, None if weights is None else weights.numpy(), threshold)
    for name, a, b in zip(("offsets", "slots", "rows"), got, want):
        assert np.array_equal(a, b), name


@pytest.mark.parametrize("T,k,E", [
    (1, 1, 1), (1, 16, 1024), (1, 8, 256), (63, 1, 7), (64, 1, 64), (65, 1, 65), (16, 16, 255),
    (128, 8, 384), (129, 8, 384), (333, 4, 60), (1025, 1, 1000), (700, 6, 1024), (2049, 8, 128),
    (9000, 8, 384), (70001, 1, 100), (20000, 16, 3)])
def test_sort_matches_the_definition(cl, T, k, E):
    g = gen(T + E)
    check_sort(cl, some_ids(g, T, k, E, padded=T // 10), E)
    w = torch.rand((T, k), generator=g)
    w[::5] = NAN  # (a NaN weight is not below the threshold)
    check_sort(cl, some_ids(g, T, k, E), E, w, 0.3)


@pytest.mark.parametrize("T,k,E", [(5, 2, 3), (300, 8, 60), (5000, 4, 1024)])
def test_sort_one_group_or_none(cl, T, k, E):
    check_sort(cl, torch.full((T, k), -1, dtype=torch.int32), E)
    check_sort(cl, torch.full((T, k), E - 1, dtype=torch.int32), E)
    check_sort(cl, torch.zeros((T, k), dtype=torch.int32), E)
    check_sort(cl, torch.zeros((T, k), dtype=torch.int32), E, torch.zeros((T, k)), 1.0)


def test_sort_no_tokens_and_refusals(cl):
    e = torch.empty((0, 4), dtype=torch.int32, device="cuda")
    off = torch.full((9,), 5, dtype=torch.int32, device="cuda")
    cl.sort_tokens(e, 4, 8, off, e, e)
    assert off.tolist() == [0] * 9
    i = torch.zeros((6, 2), dtype=torch.int32, device="cuda")
    for bad in (dict(top_k=5), dict(top_k=17), dict(n_experts=0), dict(n_experts=9), dict(slots=i[:5]),
                dict(rows=i.long()), dict(ids=i.t()), dict(weights=i), dict(offsets=off[:8])):
        a = dict(ids=i, top_k=2, n_experts=8, offsets=off, slots=i, rows=i)
        a.update(bad)
        with pytest.raises(ValueError):
            cl.sort_tokens(**a)
    ws = torch.empty(64, dtype=torch.uint8, device="cuda")
    big = torch.zeros(65536, dtype=torch.int32, device="cuda")
    assert cl.sort_tokens_workspace_bytes(65536, 1, 8) > 64
    with pytest.raises(ValueError):
        cl.sort_tokens(big, 1, 8, off, big.clone(), big.clone(), workspace=ws)


def test_sort_over_a_workspace_and_the_librarys(cl):
    for T, k, E in ((3000, 8, 384), (40000, 4, 17), (10, 2, 4)):
        ids = some_ids(gen(T), T, k, E)
        ws = torch.empty(max(16, cl.sort_tokens_workspace_bytes(T + 5000, k, E)), dtype=torch.uint8,
                         device="cuda")
        ws.fill_(255)
        for a, b in zip(run_sort(cl, ids, E, workspace=ws), run_sort(cl, ids, E)):
            assert np.array_equal(a, b)


# ---------------------------------------------------------------------------
# rows
# ---------------------------------------------------------------------------

def normal(g, shape, dtype):
    if dtype is FP8:
        return (torch.randn(shape, generator=g) * 100).to(FP8)
    return torch.randn(shape, generator=g).to(dtype)


def host(t):
    if t.dtype is FP8:
        return t.cpu().view(torch.uint8).numpy()
    return t.cpu().double().numpy()


def placed(t, at):
    """t on the device, its first value `at` values past 16 bytes."""
    buf = torch.zeros(t.numel() + at + 16, dtype=t.dtype, device="cuda")
    view = buf[at:at + t.numel()].view(t.shape)
    view.copy_(t)
    return view


def same(a, b):
    return np.array_equal(a, b, equal_nan=a.dtype.kind == "f")


COLS = [1, 2, 7, 8, 15, 16, 17, 100, 1024, 2049, 7168]
PAIRS = [(BF16, BF16), (F32, F32), (F32, BF16), (BF16, F32)]


@pytest.mark.parametrize("x_type,y_type", PAIRS + [(FP8, FP8)])
@pytest.mark.parametrize("cols", COLS)
def test_gather_and_its_gradient(cl, x_type, y_type, cols):
    for T, k, E, at in ((1, 1, 1, 0), (5, 3, 4, 1), (37, 16, 60, 3), (64, 8, 9, 8)):
        g = gen(T * cols)
        ids = some_ids(g, T, k, E, padded=T // 8)
        rows = ref.sort(ids.numpy(), E)[2]
        x = normal(g, (T, cols), x_type)
        before = normal(g, (T * k, cols), y_type)
        xd, xs = placed(x, at), placed(before, at)
        r = torch.from_numpy(rows).cuda()
        cl.gather_tokens(xd, r, xs, top_k=k)
        want = ref.gather(host(x if x_type is FP8 else x.to(y_type)), rows, host(before))
        assert same(host(xs), want)
        if x_type is FP8:
            continue
        # the way back, without weights: dxs of x's type into dx of y's
        dxs = normal(g, (T * k, cols), x_type)
        left = np.ones(T * k, bool)
        left[rows[rows >= 0]] = False
        dxs[torch.from_numpy(left)] = NAN
        dx = placed(torch.full((T, cols), NAN, dtype=y_type), at)
        cl.gather_tokens_grad(placed(dxs, at), r, dx, top_k=k)
        out, bound = ref.combine(host(dxs), rows, None, None, y_type is BF16)
        assert np.all(np.abs(host(dx) - out) <= bound)


@pytest.mark.parametrize("y_type,out_type", PAIRS)
@pytest.mark.parametrize("cols", COLS)
def test_combine(cl, y_type, out_type, cols):
    for T, k, E, at in ((1, 1, 1, 0), (3, 16, 16, 1), (50, 6, 60, 5), (33, 9, 40, 8)):
        g = gen(T + cols)
        ids = some_ids(g, T, k, E, padded=T // 8)
        rows = ref.sort(ids.numpy(), E)[2]
        ys = normal(g, (T * k, cols), y_type)
        w = torch.rand((T, k), generator=g) * 2 - 0.5
        left = np.ones(T * k, bool)
        left[rows[rows >= 0]] = False
        ys[torch.from_numpy(left)] = NAN     # rows that no slot has
        w[torch.from_numpy(rows < 0)] = NAN  # weights of slots left out
        res = normal(g, (T, cols), out_type)
        r = torch.from_numpy(rows).cuda()
        for weights, residual, inplace in ((w, res, False), (w, res, True), (w, None, False),
                                           (None, res, False)):
            out = placed(res if inplace else torch.full((T, cols), NAN, dtype=out_type), at)
            rd = None if residual is None else out if inplace else placed(res, at)
            cl.combine_tokens(placed(ys, at), r, out, top_k=k, residual=rd,
                              weights=None if weights is None else weights.cuda())
            want, bound = ref.combine(host(ys), rows, None if weights is None else weights.numpy(),
                                      None if residual is None else host(res), out_type is BF16)
            assert np.all(np.abs(host(out) - want) <= bound)


@pytest.mark.parametrize("y_type,d_type", PAIRS)
@pytest.mark.parametrize("cols", COLS)
def test_combine_grad(cl, y_type, d_type, cols):
    for T, k, E, at in ((1, 1, 1, 0), (3, 16, 16, 1), (50, 6, 60, 5), (33, 9, 40, 8)):
        g = gen(T + cols + 1)
        ids = some_ids(g, T, k, E, padded=T // 8)
        rows = ref.sort(ids.numpy(), E)[2]
        ys, dout = normal(g, (T * k, cols), y_type), normal(g, (T, cols), d_type)
        w = torch.rand((T, k), generator=g) * 2 - 0.5
        w[torch.from_numpy(rows < 0)] = NAN
        left = np.ones(T * k, bool)
        left[rows[rows >= 0]] = False
        ys[torch.from_numpy(left)] = NAN
        before = normal(g, (T * k, cols), y_type)
        r = torch.from_numpy(rows).cuda()
        for inplace in (False, True):
            yd = placed(ys, at)
            dys = yd if inplace else placed(before, at)
            dw = torch.full((T, k), NAN, device="cuda")
            cl.combine_tokens_grad(placed(dout, at), yd, r, w.cuda(), dys, dw, top_k=k)
            want, bound, ww, wb = ref.combine_grad(host(dout), host(ys), rows, w.numpy(),
                                                   host(ys if inplace else before), y_type is BF16)
            got = host(dys)
            assert same(got[left], want[left])  # left as they were
            assert np.all(np.abs(got - want)[~left] <= bound[~left])
            assert np.all(np.abs(dw.double().cpu().numpy() - ww) <= wb)


def test_rows_with_infinities_and_large_values(cl):
    """Infinities and NaN of a slot reach its own token only; bf16 rounding at the top."""
    small = torch.tensor([[1e-40, -3e-39, 1.4e-45, 9.2e-41, 4.6e-41, 1.1754944e-38, -1e-45, 0.0]])
    r = torch.tensor([[0, 1]], dtype=torch.int32).cuda()
    for t in (F32, BF16):  # subnormal values stay
        xs = torch.empty((2, 8), dtype=t, device="cuda")
        cl.gather_tokens(small.cuda(), r, xs, top_k=2)
        assert same(host(xs), small.to(t).double().expand(2, 8).numpy())
        out = torch.empty((1, 8), dtype=t, device="cuda")
        cl.combine_tokens(xs, r, out, top_k=2, weights=torch.tensor([[1.0, 0.0]]).cuda())
        assert same(host(out), small.to(t).double().numpy())
    x = torch.tensor([[float("inf"), -float("inf"), NAN, 3.4e38, 3.3895e38, -3.4e38, 1e-45, -0.0]])
    rows = torch.tensor([[1, 0]], dtype=torch.int32).cuda()
    for t in (F32, BF16):
        xs = torch.empty((2, 8), dtype=t, device="cuda")
        cl.gather_tokens(x.cuda(), rows, xs, top_k=2)
        want = x.to(t).double().expand(2, 8).numpy()
        assert same(host(xs), want)
    ys = torch.zeros((4, 8))
    ys[0], ys[1], ys[2, 0], ys[3] = 1.0, 2.0, float("inf"), NAN
    rows = torch.tensor([[0, 2], [1, -1]], dtype=torch.int32).cuda()
    out = torch.empty((2, 8), device="cuda")
    cl.combine_tokens(ys.cuda(), rows, out, top_k=2)
    assert out.tolist() == [[float("inf")] + [1.0] * 7, [2.0] * 8]


def test_row_numbers_out_of_range_are_left_out(cl):
    """Row numbers that sort_tokens never gives touch nothing."""
    T, k, cols = 3, 2, 24
    rows = torch.tensor([[0, 6], [2 ** 31 - 1, -2 ** 31], [5, -1]], dtype=torch.int32).cuda()
    x = torch.randn((T, cols), generator=gen(1)).cuda()
    xs = torch.zeros((T * k, cols), device="cuda")
    cl.gather_tokens(x, rows, xs, top_k=k)
    assert torch.equal(xs[0], x[0]) and torch.equal(xs[5], x[2]) and not xs[1:5].any()
    out = torch.empty_like(x)
    cl.gather_tokens_grad(xs, rows, out, top_k=k)
    assert torch.equal(out[0], x[0]) and not out[1].any() and torch.equal(out[2], x[2])
    dw, dys = torch.empty((T, k), device="cuda"), torch.zeros_like(xs)
    cl.combine_tokens_grad(x, xs, rows, torch.ones((T, k), device="cuda"), dys, dw, top_k=k)
    assert torch.equal(dys[0], x[0]) and not dys[1:5].any()
    assert dw[0, 1] == 0 and dw[1].tolist() == [0, 0] and dw[2, 1] == 0


def test_moves_of_nothing_and_refusals(cl):
    e = torch.empty((0, 2), dtype=torch.int32, device="cuda")
    x = torch.empty((0, 16), device="cuda")
    cl.gather_tokens(x, e, x, top_k=2)
    cl.combine_tokens(x, e, x, top_k=2)
    cl.combine_tokens_grad(x, x, e, torch.empty((0, 2), device="cuda"), x,
                           torch.empty((0, 2), device="cuda"), top_k=2)
    r = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    x, y, w = (torch.zeros(s, device="cuda") for s in ((3, 16), (6, 16), (3, 2)))
    h = y.half()
    for f in (lambda: cl.gather_tokens(x, r, y[:5], top_k=2), lambda: cl.gather_tokens(x, r, h, top_k=2),
              lambda: cl.gather_tokens(x.to(FP8), r, y, top_k=2),
              lambda: cl.gather_tokens(x.t(), r, y, top_k=2),
              lambda: cl.gather_tokens(x, r.long(), y, top_k=2),
              lambda: cl.gather_tokens(x[:, :0], r, y[:, :0], top_k=2),
              lambda: cl.gather_tokens(x, r, y, top_k=4), lambda: cl.gather_tokens(x, r, y, top_k=0),
              lambda: cl.combine_tokens(y, r, x.half(), top_k=2),
              lambda: cl.combine_tokens(y, r, x, top_k=2, weights=w[:2]),
              lambda: cl.combine_tokens(y, r, x, top_k=2, residual=x.bfloat16()),
              lambda: cl.combine_tokens(y, r, y, top_k=2),
              lambda: cl.combine_tokens_grad(x, y, r, w, y.bfloat16(), w, top_k=2),
              lambda: cl.combine_tokens_grad(x, y, r, w, y, w.double(), top_k=2),
              lambda: cl.combine_tokens_grad(y, y, r, w, y, w, top_k=2)):
        with pytest.raises(ValueError):
            f()


def test_offsets_past_32_bits(cl):
    """Rows whose values lie more than 2^32 bytes, and 2^31 values, into a buffer."""
    T, k, cols = 147456, 16, 1024
    g = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.arange(k, dtype=torch.int32, device="cuda").expand(T, k).contiguous()
    off, slots, rows = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (k + 1, T * k, T * k))
    cl.sort_tokens(ids, k, k, off, slots, rows)
    x = torch.randn((T, cols), generator=g, device="cuda").bfloat16()
    xs = torch.empty((T * k, cols), dtype=BF16, device="cuda")
    assert xs.numel() > 2 ** 31
    cl.gather_tokens(x, rows.view(T, k), xs, top_k=k)
    for e in range(k):
        assert torch.equal(xs[e * T:(e + 1) * T], x)
    w = torch.zeros((T, k), device="cuda")
    w[:, k - 1] = 1.0
    out = torch.empty_like(x)
    cl.combine_tokens(xs, rows.view(T, k), out, top_k=k, weights=w)
    assert torch.equal(out, x)
    dw = torch.empty_like(w)
    cl.combine_tokens_grad(x, xs, rows.view(T, k), w, xs, dw, top_k=k)
    assert torch.equal(xs[(k - 1) * T:], x) and not xs[:(k - 1) * T].any()
    assert torch.equal(dw[:, 0], dw[:, k - 1]) and bool((dw > 0).all())


def test_repeats_streams_and_recorded_calls(cl):
    """The same bits on every run, on another stream, and from a replayed graph."""
    T, k, E, cols = 3000, 8, 384, 520
    g = gen(9)
    ids = [some_ids(g, T, k, E, padded=17).cuda() for _ in range(2)]
    w = torch.rand((T, k), generator=g).cuda()
    x, dout = (torch.randn((T, cols), generator=g).bfloat16().cuda() for _ in range(2))
    ws = torch.empty(cl.sort_tokens_workspace_bytes(T, k, E), dtype=torch.uint8, device="cuda")
    idb = ids[0].clone()

    def buffers():
        i = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (E + 1, T * k, T * k)]
        return i + [torch.zeros((T * k, cols), dtype=BF16, device="cuda"), torch.zeros_like(x),
                    torch.zeros((T * k, cols), dtype=BF16, device="cuda"), torch.zeros_like(w)]

    def call(b):
        off, slots, rows, xs, out, dys, dw = b
        cl.sort_tokens(idb, k, E, off, slots, rows, weights=w, threshold=0.05, workspace=ws)
        cl.gather_tokens(x, rows, xs, top_k=k)
        cl.combine_tokens(xs, rows, out, top_k=k, weights=w, residual=x)
        cl.combine_tokens_grad(dout, xs, rows, w, dys, dw, top_k=k)

    want = []
    for i in range(2):
        idb.copy_(ids[i])
        want.append(buffers())
        call(want[i])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = buffers()
        call(b)
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(b, want[1]))
    b = buffers()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(b)
    for i in (0, 1, 1, 0):
        idb.copy_(ids[i])
        for t in b:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        call(buffers())  # eager work of the same kind in between
        assert all(torch.equal(p, q) for p, q in zip(b, want[i]))
