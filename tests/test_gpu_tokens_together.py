"""Routing, sorting, experts run one by one, and back, as a caller would; with the
adapters of many requests beside shared projections; and the gradients of a whole
step against differences of its 64-bit value."""
import numpy as np
import pytest
import torch

import tokens_ref as ref
from conftest import rel_l2
from test_gpu_adapters import cl, gen, host, plan  # noqa: F401

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def sorted_by_expert(cl, ids, E):
    T, k = ids.shape
    out = [torch.empty(n, dtype=torch.int32, device="cuda") for n in (E + 1, T * k)]
    rows = torch.empty((T, k), dtype=torch.int32, device="cuda")
    cl.sort_tokens(ids, k, E, *out, rows)
    return out[0], out[1], rows


def test_experts_one_by_one(cl):
    """route_experts, sort, gather, expert_forward on each expert's rows, combine: each
    token's weighted sum of its own experts' outputs."""
    T, H, I, E, k, G = 45, 256, 128, 12, 3, 32
    g = gen(31)
    from cascadia_amd import api

    per = api.expert_bytes(H, I, G)
    flat = torch.randint(0, 256, (E, per), generator=g, dtype=torch.uint8)
    sizes = api._section_sizes(H, I, G, cl.TILING_CRATE)
    at = np.cumsum([0] + sizes)
    for s in (1, 3, 5):
        n = sizes[s] // 2
        sc = (torch.rand((E, n), generator=g) * 0.02 + 0.005).to(BF16)
        flat[:, at[s]:at[s + 1]] = sc.view(torch.uint8).view(E, -1)
    weights = [cl.ExpertWeights(flat[e].cuda(), H, I, G, cl.SCALE_BF16) for e in range(E)]
    logits = torch.randn((T, E), generator=g).cuda()
    ids = torch.empty((T, k), dtype=torch.int32, device="cuda")
    w = torch.empty((T, k), device="cuda")
    cl.route_experts(logits, k, ids, w)
    ids[-2:] = -1  # padding
    x = torch.randn((T, H), generator=g).cuda()
    off, slots, rows = sorted_by_expert(cl, ids, E)
    xs = torch.zeros((T * k, H), dtype=BF16, device="cuda")
    cl.gather_tokens(x, rows, xs, top_k=k)
    ys = torch.zeros_like(xs)
    ends = off.tolist()
    for e in range(E):
        if ends[e + 1] > ends[e]:
            part = slice(ends[e], ends[e + 1])
            cl.expert_forward(xs[part], *weights[e].slices(), ys[part], group_size=G,
                              scale_dtype=cl.SCALE_BF16)
    out = torch.empty_like(x)
    cl.combine_tokens(ys, rows, out, top_k=k, weights=w, residual=x)
    # the same experts' outputs, slot by slot
    want, bound = ref.combine(host(ys), rows.cpu().numpy(), w.cpu().numpy(), host(x), False)
    assert np.all(np.abs(host(out) - want) <= bound)
    # each token's own rows went through its own experts
    one = torch.empty((1, H), dtype=BF16, device="cuda")
    for t, j in ((0, 0), (7, 2), (42, 1)):
        e = int(ids[t, j])
        cl.expert_forward(x[t:t + 1].to(BF16).contiguous(), *weights[e].slices(), one, group_size=G,
                          scale_dtype=cl.SCALE_BF16)
        assert rel_l2(host(ys[rows[t, j]]), host(one[0])) < 1e-2
    assert torch.equal(out[-2:], x[-2:])


@pytest.mark.parametrize("T", [1, 40, 200])
def test_adapters_beside_the_projections(cl, T):
    """One grouping of a batch's rows beside an INT4 and an e4m3 projection."""
    K, N, E, R = 512, 384, 9, 16
    g = gen(32)
    wb = (torch.randn((N, K), generator=g) / K ** 0.5).to(BF16).cuda()
    packed, sc = cl.quantize_int4_group(wb, N, K, 32)
    codes, cs = cl.quantize_fp8_blocks(wb, N, K)
    a = (torch.randn((E, R, K), generator=g) / K ** 0.5).to(BF16)
    b = (torch.randn((E, N, R), generator=g) * 0.1).to(BF16)
    A = cl.Adapters(a.cuda(), b.cuda())
    ids = torch.randint(-1, E, (T,), generator=g, dtype=torch.int32)
    ids[0] = 4
    off, slots = plan(cl, ids, E)
    x = torch.randn((T, K), generator=g).to(BF16)
    for int4 in (True, False):
        base = torch.empty((T, N), device="cuda")
        if int4:
            cl.dequant_gemm_int4_multi_auto(packed, sc, x.cuda(), N, K, T, base, group_size=32,
                                            scale_dtype=cl.SCALE_BF16)
        else:
            cl.fp8_gemm(codes, cs, x.cuda(), N, K, T, base)
        for y_type in (F32, BF16):
            y = torch.empty((T, N), dtype=y_type, device="cuda")
            cl.adapters_forward(A, x.cuda(), off, slots, y, base=base)
            want, bound = ref.adapters(host(a), host(b), [R] * E, [1.0] * E, ids.tolist(), host(x),
                                       host(base), y_type is BF16)
            assert np.all(np.abs(host(y) - want) <= bound)


def test_gradients_of_a_step(cl):
    """x -> gather -> (ys = c * xs^2) -> combine -> <., dout>: the gradients of x and of
    the weights through combine_tokens_grad and gather_tokens_grad against central
    differences of the same value in 64 bits."""
    T, H, E, k = 12, 40, 5, 2
    g = gen(33)
    ids = torch.rand((T, E), generator=g).topk(k, 1).indices.int()
    ids[3] = -1
    off, slots, rows = sorted_by_expert(cl, ids.cuda(), E)
    r = rows.cpu().numpy()
    x, dout = torch.randn((T, H), generator=g), torch.randn((T, H), generator=g)
    w = torch.rand((T, k), generator=g)
    c = torch.randn((T * k, H), generator=g)
    xs = torch.zeros((T * k, H), device="cuda")
    cl.gather_tokens(x.cuda(), rows, xs, top_k=k)
    ys = c.cuda() * xs * xs
    dys, dw = torch.zeros_like(ys), torch.empty((T, k), device="cuda")
    cl.combine_tokens_grad(dout.cuda(), ys, rows, w.cuda(), dys, dw, top_k=k)
    dx = torch.empty((T, H), device="cuda")
    cl.gather_tokens_grad(dys * 2 * c.cuda() * xs, rows, dx, top_k=k)

    def value(x, w):
        s = ref.gather(x, r, np.zeros((T * k, H)))
        return (ref.combine(host(c) * s * s, r, w, None, False)[0] * host(dout)).sum()

    x64, w64, h = host(x), host(w), 1e-5
    for t, j in ((0, 0), (3, 7), (5, 39), (11, 20)):
        d = np.zeros_like(x64)
        d[t, j] = h
        # (the value is a square in x: its central difference is off by 64-bit rounding
        # alone, 2^-52 * T * H terms of at most 60 or so, over 2 h: below 1e-6; the
        # kernels' dx is a sum of k terms 2 w c x dout, each of six roundings of 2^-24)
        diff = (value(x64 + d, w64) - value(x64 - d, w64)) / (2 * h)
        terms = sum(abs(2 * w64[t, i] * float(c[r[t, i], j]) * x64[t, j] * float(dout[t, j]))
                    for i in range(k) if r[t, i] >= 0)
        assert abs(diff - float(dx[t, j])) <= 8 * ref.U32 * terms + 1e-6
    for t, j in ((0, 0), (3, 1), (11, 1)):
        d = np.zeros_like(w64)
        d[t, j] = h
        diff = (value(x64, w64 + d) - value(x64, w64 - d)) / (2 * h)
        # (a sum of H terms c x^2 dout, three roundings each and one per addition)
        terms = 0.0 if r[t, j] < 0 else np.abs(host(c)[r[t, j]] * x64[t] ** 2 * host(dout)[t]).sum()
        assert abs(diff - float(dw[t, j])) <= (H + 4) * ref.U32 * terms + 1e-6
