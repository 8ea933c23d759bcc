"""Refusals of the token-sorting and adapter entry points, and the 64-bit reference of
their tests, on the CPU: no call here reaches the device."""
import ctypes as C

import numpy as np
import pytest
import torch

import tokens_ref as ref

P = 1 << 20  # an address that no call may read


@pytest.fixture(scope="module")
def cl():
    import cascadia_amd

    return cascadia_amd


def test_sort_refusals(cl):
    L, arg, nul = cl.lib(), cl._lib.ERR_ARG, cl._lib.ERR_NULL

    def call(ids=P, w=None, T=4, k=2, E=8, off=P, slots=P, rows=P, ws=None):
        return L.cascadia_int4_sort_tokens(ids, w, 0.0, T, k, E, off, slots, rows, ws, None)

    for kw in (dict(ids=None), dict(off=None), dict(slots=None), dict(rows=None),
               dict(T=0, off=None)):
        assert call(**kw) == nul, kw
    for kw in (dict(k=0), dict(k=17), dict(E=0), dict(E=1025), dict(T=(1 << 20) + 1), dict(ids=P + 2),
               dict(w=P + 1), dict(off=P + 2), dict(slots=P + 2), dict(rows=P + 1), dict(ws=P + 8),
               dict(T=0xFFFFFFFF)):
        assert call(**kw) == arg, kw
    need = L.cascadia_int4_sort_tokens_workspace_bytes
    for a in ((4, 0, 8), (4, 17, 8), (4, 2, 0), (4, 2, 1025), ((1 << 20) + 1, 1, 8)):
        assert need(*a) == 0
    sizes = [need(t, 8, 384) for t in range(0, 12000, 7)]
    assert sizes == sorted(sizes) and sizes[-1] > 0


def test_move_refusals(cl):
    L, arg, nul, ok = cl.lib(), cl._lib.ERR_ARG, cl._lib.ERR_NULL, cl._lib.OK

    def gather(x=P, xt=0, rows=P, T=4, k=2, cols=16, xs=P, yt=0):
        return L.cascadia_int4_gather_tokens(x, xt, rows, T, k, cols, xs, yt, None)

    for kw in (dict(x=None), dict(rows=None), dict(xs=None)):
        assert gather(**kw) == nul, kw
    for kw in (dict(k=0), dict(k=17), dict(cols=0), dict(cols=(1 << 20) + 1), dict(xt=3), dict(yt=3),
               dict(xt=2), dict(yt=2), dict(xt=1, yt=2), dict(x=P + 1), dict(xs=P + 1),
               dict(xt=1, x=P + 2), dict(yt=1, xs=P + 2), dict(rows=P + 2), dict(T=(1 << 20) + 1)):
        assert gather(**kw) == arg, kw
    assert gather(T=0, x=None, rows=None, xs=None) == ok

    def combine(ys=P, yf=0, rows=P, w=None, res=None, T=4, k=2, cols=16, out=P, of=0):
        return L.cascadia_int4_combine_tokens(ys, yf, rows, w, res, T, k, cols, out, of, None)

    for kw in (dict(ys=None), dict(rows=None), dict(out=None)):
        assert combine(**kw) == nul, kw
    for kw in (dict(k=0), dict(k=17), dict(cols=0), dict(cols=(1 << 20) + 1), dict(yf=2), dict(of=2),
               dict(ys=P + 1), dict(yf=1, ys=P + 2), dict(out=P + 1), dict(of=1, out=P + 2),
               dict(res=P + 1), dict(of=1, res=P + 2), dict(w=P + 2), dict(rows=P + 2),
               dict(T=(1 << 20) + 1)):
        assert combine(**kw) == arg, kw
    assert combine(T=0, ys=None, rows=None, out=None) == ok

    def grad(d=P, df=0, ys=P, yf=0, rows=P, w=P, T=4, k=2, cols=16, dys=P, dw=P):
        return L.cascadia_int4_combine_tokens_grad(d, df, ys, yf, rows, w, T, k, cols, dys, dw, None)

    for kw in (dict(d=None), dict(ys=None), dict(rows=None), dict(w=None), dict(dys=None),
               dict(dw=None)):
        assert grad(**kw) == nul, kw
    for kw in (dict(k=0), dict(k=17), dict(cols=0), dict(cols=(1 << 20) + 1), dict(df=2), dict(yf=2),
               dict(d=P + 1), dict(df=1, d=P + 2), dict(ys=P + 1), dict(yf=1, dys=P + 2),
               dict(dys=P + 1), dict(w=P + 2), dict(dw=P + 2), dict(rows=P + 2),
               dict(T=(1 << 20) + 1)):
        assert grad(**kw) == arg, kw
    assert grad(T=0, d=None, ys=None, rows=None, w=None, dys=None, dw=None) == ok


def test_adapters_refusals(cl):
    L, arg, nul, ok = cl.lib(), cl._lib.ERR_ARG, cl._lib.ERR_NULL, cl._lib.OK
    Set = cl._lib.AdapterSet

    def call(off=P, slots=P, x=P, xf=0, ldx=None, base=None, bf=0, ldb=0, T=4, y=2 * P, yf=0,
             ldy=None, ws=None, **kw):
        a = dict(k_cols=64, n_rows=48, max_rank=16, n_adapters=4, a=P, b=P, ranks=None, scales=None)
        a.update(kw)
        ldx = a["k_cols"] if ldx is None else ldx
        ldy = a["n_rows"] if ldy is None else ldy
        return L.cascadia_int4_adapters_forward(C.byref(Set(**a)), off, slots, x, xf, ldx, base, bf,
                                                ldb, T, y, yf, ldy, ws, None)

    assert L.cascadia_int4_adapters_forward(None, P, P, P, 0, 64, None, 0, 0, 4, P, 0, 48, None,
                                            None) == nul
    for kw in (dict(a=None), dict(b=None), dict(off=None), dict(slots=None), dict(x=None),
               dict(y=None)):
        assert call(**kw) == nul, kw
    for kw in (dict(k_cols=0), dict(k_cols=60), dict(k_cols=(1 << 20) + 8), dict(n_rows=0),
               dict(n_rows=(1 << 22) + 1), dict(max_rank=0), dict(max_rank=12), dict(max_rank=264),
               dict(n_adapters=0), dict(n_adapters=1025), dict(a=P + 8), dict(b=P + 8),
               dict(ranks=P + 2), dict(scales=P + 2), dict(T=(1 << 20) + 1), dict(xf=2), dict(bf=2),
               dict(yf=2), dict(ldx=63), dict(ldy=47), dict(base=P, ldb=47), dict(ldx=(1 << 29) + 1),
               dict(ldy=(1 << 29) + 1), dict(base=P, ldb=(1 << 29) + 1), dict(off=P + 2), dict(slots=P + 2),
               dict(x=P + 1), dict(xf=1, x=P + 2), dict(y=P + 1), dict(yf=1, y=P + 2),
               dict(base=P + 1, ldb=48), dict(base=P + 2, bf=1, ldb=48), dict(ws=P + 8),
               dict(base=2 * P, ldb=49), dict(base=2 * P, bf=1, ldb=48)):
        assert call(**kw) == arg, kw
    assert call(T=0, off=None, slots=None, x=None, y=None) == ok
    need = L.cascadia_int4_adapters_workspace_bytes
    assert need(C.byref(Set(64, 48, 12, 4, P, P, None, None)), 4) == 0
    for k, r, e in ((4096, 16, 100), (64, 256, 1), (14336, 64, 1024), (200, 8, 3)):
        s = Set(k, 48, r, e, P, P, None, None)
        sizes = [need(C.byref(s), t) for t in range(1, 3000)]
        assert sizes == sorted(sizes) and sizes[0] > 0, (k, r, e)


def test_host_tensors_are_refused(cl):
    i, f = torch.zeros((4, 1), dtype=torch.int32), torch.zeros((4, 8))
    w = torch.zeros((4, 1))
    h = torch.zeros((1, 8, 8), dtype=torch.bfloat16)
    for call in (lambda: cl.sort_tokens(i, 1, 3, i, i, i), lambda: cl.gather_tokens(f, i, f, top_k=1),
                 lambda: cl.combine_tokens(f, i, f, top_k=1),
                 lambda: cl.gather_tokens_grad(f, i, f, top_k=1),
                 lambda: cl.combine_tokens_grad(f, f, i, w, f, w, top_k=1),
                 lambda: cl.Adapters(h, h)):
        with pytest.raises(ValueError):
            call()


# ---- the reference itself ----

def test_reference_sort_by_hand():
    ids = np.array([[2, 0], [-1, 2], [0, 5], [1, 2]])
    off, slots, rows = ref.sort(ids, 4)
    assert off.tolist() == [0, 2, 3, 6, 6] and slots.tolist() == [1, 4, 6, 0, 3, 7, 2, 5]
    assert rows.tolist() == [[3, 0], [-1, 4], [1, -1], [2, 5]]
    w = np.array([[0.5, 0.1], [1, 1], [1, 1], [np.nan, 0.1]])
    off, slots, rows = ref.sort(ids, 4, w, 0.2)
    assert off.tolist() == [0, 1, 2, 4, 4] and slots.tolist() == [4, 6, 0, 3, 1, 2, 5, 7]
    assert rows.tolist() == [[2, -1], [-1, 3], [0, -1], [1, -1]]


def test_reference_gradients_are_differences():
    """<combine's output, dout> changes with ys and the weights as the gradients say."""
    g = np.random.default_rng(4)
    ids = np.array([[0, 2], [1, -1], [2, 0]])
    rows = ref.sort(ids, 3)[2]
    ys, w = g.standard_normal((6, 5)), g.random((3, 2))
    dout, res = g.standard_normal((3, 5)), g.standard_normal((3, 5))
    dys, _, dw, _ = ref.combine_grad(dout, ys, rows, w, np.zeros((6, 5)), False)

    def loss(ys, w):
        return (ref.combine(ys, rows, w, res, False)[0] * dout).sum()

    for at in np.ndindex(ys.shape):
        d = np.zeros_like(ys)
        d[at] = 1e-4
        assert abs((loss(ys + d, w) - loss(ys - d, w)) / 2e-4 - dys[at]) < 1e-8
    for at in np.ndindex(w.shape):
        d = np.zeros_like(w)
        d[at] = 1e-4
        assert abs((loss(ys, w + d) - loss(ys, w - d)) / 2e-4 - dw[at]) < 1e-8
    # and gather's: <xs, dxs> changes with x as combine without weights says
    dxs = g.standard_normal((6, 5))
    x = g.standard_normal((3, 5))
    dx = ref.combine(dxs, rows, None, None, False)[0]
    for at in np.ndindex(x.shape):
        d = np.zeros_like(x)
        d[at] = 1e-4
        up, down = (ref.gather(x + s * d, rows, np.zeros((6, 5))) for s in (1, -1))
        assert abs(((up - down) * dxs).sum() / 2e-4 - dx[at]) < 1e-8


def test_reference_adapters_against_loops():
    g = np.random.default_rng(5)
    a, b = g.integers(-3, 4, (2, 8, 16)) * 1.0, g.integers(-3, 4, (2, 5, 8)) * 1.0
    x, base = g.integers(-3, 4, (3, 16)) * 1.0, g.integers(-3, 4, (3, 5)) * 1.0
    y, bound = ref.adapters(a, b, [3, 8], [0.5, 2.0], [1, -1, 0], x, base, False)
    for t, (i, r, s) in enumerate(((1, 8, 2.0), (0, 0, 0.0), (0, 3, 0.5))):
        for n in range(5):
            d = sum(b[i, n, j] * sum(a[i, j, c] * x[t, c] for c in range(16)) for j in range(r))
            assert y[t, n] == base[t, n] + s * d
    assert np.all(bound[1] <= 4 * ref.U32 * np.abs(base[1]) + 1e-30)
