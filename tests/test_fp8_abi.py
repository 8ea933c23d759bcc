"""Refusals of the routing and 8-bit floating-point entry points, and the 64-bit
reference of their tests, on the CPU: no call here reaches the device."""
import ctypes as C

import numpy as np
import pytest
import torch

import fp8_ref as ref

P = 1 << 20  # an address that no call may read


@pytest.fixture(scope="module")
def cl():
    import cascadia_amd

    return cascadia_amd


def test_router_refusals(cl):
    f = cl.lib().cascadia_int4_route_experts
    Router = cl._lib.Router

    def call(T=4, logits=P, bf16=0, ids=P, w=P, **kw):
        a = dict(n_experts=64, top_k=4, score=1, n_groups=1, top_groups=1, group_best=1, normalize=1,
                 scale=1.0, bias=None)
        a.update(kw)
        return f(C.byref(Router(**a)), logits, bf16, T, ids, w, None)

    arg, nul = cl._lib.ERR_ARG, cl._lib.ERR_NULL
    assert f(None, P, 0, 4, P, P, None) == nul
    for kw in (dict(logits=None), dict(ids=None), dict(w=None)):
        assert call(**kw) == nul
    for kw in (dict(n_experts=0), dict(n_experts=1025), dict(top_k=0), dict(top_k=17),
               dict(n_experts=3), dict(score=2), dict(n_groups=0), dict(n_groups=65),
               dict(n_groups=5), dict(n_groups=4, top_groups=0), dict(n_groups=4, top_groups=5),
               dict(n_groups=32, top_groups=1), dict(group_best=0), dict(group_best=3),
               dict(bf16=2), dict(logits=P + 2), dict(logits=P + 1, bf16=1), dict(ids=P + 2),
               dict(w=P + 1), dict(bias=P + 2), dict(T=(1 << 30) + 1)):
        assert call(**kw) == arg, kw
    assert call(T=0, logits=None, ids=None, w=None) == cl._lib.OK


def test_quantize_refusals(cl):
    L, arg, nul = cl.lib(), cl._lib.ERR_ARG, cl._lib.ERR_NULL
    q, b = L.cascadia_int4_fp8_quantize, L.cascadia_int4_fp8_quantize_blocks
    for a in ((None, 0, 4, 32, P, P), (P, 0, 4, 32, None, P), (P, 0, 4, 32, P, None)):
        assert q(*a, None) == nul
    for a in ((P, 0, 4, 24, P, P), (P, 0, 4, 0, P, P), (P, 2, 4, 32, P, P), (P + 8, 0, 4, 32, P, P),
              (P, 0, 4, 32, P + 8, P), (P, 0, 4, 32, P, P + 2), (P, 0, (1 << 24) + 1, 32, P, P),
              (P, 0, 1, (1 << 20) + 16, P, P)):
        assert q(*a, None) == arg
    assert q(None, 0, 0, 32, None, None, None) == cl._lib.OK
    for a in ((None, 4, 32, P, P), (P, 4, 32, None, P), (P, 4, 32, P, None)):
        assert b(*a, None) == nul
    for a in ((P, 0, 32, P, P), (P, 4, 40, P, P), (P + 2, 4, 32, P, P), (P, 4, 32, P + 4, P),
              (P, 4, 32, P, P + 1), (P, (1 << 22) + 1, 32, P, P)):
        assert b(*a, None) == arg


def test_gemm_refusals(cl):
    L, arg, nul = cl.lib(), cl._lib.ERR_ARG, cl._lib.ERR_NULL

    def call(n=32, k=64, w=P, ws=P, x=P, xt=2, xs=P, seq=4, y=P, f32=1, buf=None):
        return L.cascadia_int4_fp8_gemm(n, k, w, ws, x, xt, xs, seq, y, f32, buf, None)

    for kw in (dict(w=None), dict(ws=None), dict(x=None), dict(xs=None), dict(y=None)):
        assert call(**kw) == nul
    for kw in (dict(n=0), dict(k=0), dict(k=72), dict(seq=0), dict(xt=3), dict(xt=0), dict(f32=2),
               dict(w=P + 8), dict(x=P + 4), dict(ws=P + 2), dict(xs=P + 2), dict(y=P + 2),
               dict(y=P + 1, f32=0), dict(buf=P + 8), dict(n=(1 << 24) + 1),
               dict(k=(1 << 20) + 16), dict(seq=(1 << 24) + 1),
               dict(seq=1 << 24, k=1 << 20)):
        assert call(**kw) == arg, kw
    need = L.cascadia_int4_fp8_gemm_workspace_bytes
    for a in ((0, 64, 0, 4), (32, 72, 0, 4), (32, 64, 3, 4), (32, 64, 0, 0)):
        assert need(*a) == 0
    assert need(32, 64, 0, 4) >= 4 * 64 + 4 * 4
    # one workspace of the largest call serves every smaller one
    for x_type in (0, 1, 2):
        for n, k in ((4096, 4096), (576, 7168), (100, 20496), (14336, 4096)):
            sizes = [need(n, k, x_type, m) for m in range(1, 600)]
            assert sizes == sorted(sizes)


def test_moe_refusals(cl):
    L, arg, nul = cl.lib(), cl._lib.ERR_ARG, cl._lib.ERR_NULL
    Layer = cl._lib.Fp8MoeLayer

    def call(k=2, ids=P, w=P, x=P, xf=0, res=None, T=4, out=P, of=0, buf=None, **kw):
        a = dict(hidden=64, inter=32, n_experts=4, gate_up=P, gate_up_scales=P, down=P,
                 down_scales=P, tiled=0)
        a.update(kw)
        return L.cascadia_int4_fp8_moe_forward(C.byref(Layer(**a)), k, ids, w, 0.0, x, xf, res, T,
                                               out, of, buf, None)

    assert L.cascadia_int4_fp8_moe_forward(None, 2, P, P, 0.0, P, 0, None, 4, P, 0, None,
                                           None) == nul
    for kw in (dict(gate_up=None), dict(gate_up_scales=None), dict(down=None),
               dict(down_scales=None), dict(ids=None), dict(w=None), dict(x=None), dict(out=None)):
        assert call(**kw) == nul, kw
    for kw in (dict(hidden=0), dict(hidden=72), dict(inter=24), dict(n_experts=0),
               dict(n_experts=1025), dict(k=0), dict(k=17), dict(T=0), dict(T=(1 << 20) + 1),
               dict(gate_up=P + 8), dict(down=P + 4), dict(gate_up_scales=P + 2), dict(xf=2),
               dict(of=2), dict(tiled=2), dict(x=P + 8), dict(out=P + 8), dict(res=P + 8), dict(buf=P + 8),
               dict(ids=P + 2), dict(w=P + 2)):
        assert call(**kw) == arg, kw
    need = L.cascadia_int4_fp8_moe_workspace_bytes
    lay = Layer(256, 128, 16, P, P, P, P, 1)
    sizes = [need(C.byref(lay), 4, t) for t in range(1, 600)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert need(C.byref(lay), 0, 4) == 0


def test_tile_refusals(cl):
    L, arg, nul = cl.lib(), cl._lib.ERR_ARG, cl._lib.ERR_NULL
    f = L.cascadia_int4_fp8_tile_weights
    assert f(1, 4, 32, None, P, None) == nul and f(1, 4, 32, P, None, None) == nul
    for a in ((0, 4, 32, P, P), (1, 0, 32, P, P), (1, 4, 40, P, P), (1, 4, 32, P + 8, P),
              (1, 4, 32, P, P + 8), ((1 << 20) + 1, 4, 32, P, P), (1 << 20, 1 << 20, 1 << 14, P, P)):
        assert f(*a, None) == arg
    b = L.cascadia_int4_fp8_tiled_bytes
    assert b(1, 16) == 128 * 128 and b(129, 272) == 2 * 3 * 128 * 128 and b(4, 40) == 0


def test_host_tensors_are_refused(cl):
    x = torch.zeros((2, 32))
    ids, w = torch.zeros((2, 1), dtype=torch.int32), torch.zeros((2, 1))
    c, s = torch.zeros((2, 32), dtype=torch.uint8), torch.zeros((2, 1))
    for f in (lambda: cl.route_experts(x, 1, ids, w), lambda: cl.quantize_fp8(x, 2, 32, c, s),
              lambda: cl.quantize_fp8_blocks(x.to(torch.bfloat16), 2, 32),
              lambda: cl.fp8_gemm(c, s, x, 2, 32, 2, x), lambda: cl.Fp8Experts(c, s, c, s, 1, 32, 16)):
        with pytest.raises(ValueError):
            f()


# ---- the reference itself ----

def test_reference_rounding_is_torchs():
    v = torch.randn(20000, generator=torch.Generator().manual_seed(1)) * 100
    v = torch.cat([v, v * 2.0 ** -12, torch.tensor([0.0, 448.0, -448.0, 2.0 ** -10])]).clamp_(-448, 448)
    assert np.array_equal(ref.round_e4m3(v.double().numpy()), ref.e4m3(v.to(torch.float8_e4m3fn)))


def test_reference_product_against_loops():
    g = np.random.default_rng(2)
    xq, wq = g.integers(-8, 8, (3, 160)) * 1.0, g.integers(-8, 8, (130, 160)) * 1.0
    xs, ws = g.random((3, 2)), g.random((2, 2))
    y, _ = ref.gemm(xq, xs, wq, ws)
    for t in range(3):
        for n in (0, 127, 128, 129):
            s = sum(xq[t, c] * wq[n, c] * xs[t, c // 128] * ws[n // 128, c // 128]
                    for c in range(160))
            assert abs(y[t, n] - s) < 1e-9


def test_reference_layer_against_a_plain_one():
    """With codes that need no rounding the layer is the textbook SwiGLU."""
    g = np.random.default_rng(3)
    E, H, I = 2, 16, 16
    gu, dn = g.integers(-4, 5, (E, 2, I, H)) * 1.0, g.integers(-4, 5, (E, H, I)) * 1.0
    gus, dns = np.full((E, 2, 1, 1), 0.01), np.full((E, 1, 1), 0.02)
    x = np.full((2, H), 448.0)
    ids, w = np.array([[0, 1], [1, -1]]), np.array([[0.5, 0.25], [1.0, 9.0]])
    out, bound = ref.moe(x, gu, gus, dn, dns, ids, w, 0.0, None)
    for t in range(2):
        want = np.zeros(H)
        for e, p in zip(ids[t], w[t]):
            if e >= 0:
                h = ref.silu(gu[e, 0] @ x[t] * 0.01) * (gu[e, 1] @ x[t] * 0.01)
                q, s = ref.quotients(h[None], 1)
                want += p * (dn[e] @ (ref.round_e4m3(q)[0] * s[0, 0]) * 0.02)
        assert np.allclose(out[t], want, rtol=1e-12) and np.all(bound[t] >= 0)


def test_reference_route_on_a_case_by_hand():
    logits = np.array([[1.0, 3.0, 2.0, 2.0, 0.0, 5.0, 4.0, -1.0]])
    ids, w = ref.route(logits, 3, "sigmoid", None, 2, 1, 1, False, 1.0)
    assert ids.tolist() == [[5, 6, 4]]
    ids, w = ref.route(logits, 3, "softmax", None, 1, 1, 1, True, 2.0)
    assert ids.tolist() == [[5, 6, 1]] and abs(w.sum() - 2.0) < 1e-12
    bias = np.array([9.0, 0, 0, 0, 0, 0, 0, 9.0])
    ids, w = ref.route(logits, 2, "sigmoid", bias, 1, 1, 1, False, 1.0)
    assert ids.tolist() == [[0, 7]] and abs(w[0, 0] - 1 / (1 + np.exp(-1.0))) < 1e-12


def test_layer_workspace_of_more_tokens_serves_fewer(cl):
    """One token keeps its slots' h in f32, more of them (here on tiles at once: one
    expert takes all 16 slots) only its codes."""
    Layer, need = cl._lib.Fp8MoeLayer, cl.lib().cascadia_int4_fp8_moe_workspace_bytes
    for hidden, inter, experts, k in ((16, 4096, 1, 16), (16, 4096, 2, 16), (32, 4096, 4, 16),
                                      (16, 2048, 3, 8), (256, 128, 1, 1)):
        lay = Layer(hidden, inter, experts, P, P, P, P, 0)
        sizes = [need(C.byref(lay), k, t) for t in range(1, 300)]
        assert sizes == sorted(sizes), (hidden, inter, experts, k)
