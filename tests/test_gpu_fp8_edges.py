"""Calls at the borders of the routing and 8-bit forms: infinite biases, rows of the
longest length that one kernel holds, one token with slots left out, scales off 16
bytes, very wide layers.  Against the 64-bit reference (fp8_ref)."""
import numpy as np
import pytest
import torch

import fp8_ref as ref
from test_gpu_fp8 import (check_gemm, check_moe, check_route, cl, gemm_case, gen, moe_case,  # noqa: F401
                          normal, run_moe, run_route)

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups,best", [(1, 1, 1), (8, 3, 2), (8, 3, 1)])
def test_route_infinite_biases(cl, score, groups, top_groups, best):
    """Experts shut off by a bias of -infinity, or chosen by +infinity."""
    g = gen(21)
    logits = normal(g, 65, 96)
    off = normal(g, 96) * 0.1
    off[torch.randperm(96, generator=g)[:40]] = -float("inf")
    check_route(cl, logits, 6, score, off, groups, top_groups, best, True, 1.5)
    most = torch.full((96,), -float("inf"))  # fewer left than are chosen
    most[[5, 50, 90]] = 0.25
    check_route(cl, logits, 6, score, most, groups, top_groups, best, True, 1.5)
    on = normal(g, 96) * 0.1
    on[[0, 17, 18, 95]] = float("inf")
    check_route(cl, logits, 6, score, on, groups, top_groups, best, False, 1.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_wide_logits(cl, score):
    """Logits far apart, whose scores underflow, and large ones close together."""
    g = gen(22)
    bias = normal(g, 64) * 2.0 ** -20
    for x in (normal(g, 33, 64) * 300, 1000 + normal(g, 33, 64), -1000 + normal(g, 33, 64) * 30,
              normal(g, 33, 64) * 1e-30, normal(g, 33, 64) * 1e37):
        for b in (None, bias):
            check_route(cl, x, 8, score, b, 1, 1, 1, False, 1.0)
            check_route(cl, x, 8, score, b, 4, 2, 2, False, 1.0)


@pytest.mark.parametrize("kind", ["fp8", "bf16", "f32"])
@pytest.mark.parametrize("m,n,k", [(1, 40, 16384), (1, 40, 16400), (7, 33, 16384), (20, 17, 16400)])
def test_gemm_longest_rows_in_lds(cl, m, n, k, kind):
    w, ws, x, xs = gemm_case(m + k, m, n, k, kind)
    for dt in (F32, BF16):
        check_gemm(cl, w, ws, x, xs, dt)


@pytest.mark.parametrize("m,n,k,form", [(5, 64, 512, 1), (40, 64, 512, 2), (65, 576, 9216, 4),
                                        (2000, 1900, 512, 3), (1700, 3600, 512, 5)])
def test_gemm_scales_off_16_bytes(cl, m, n, k, form):
    """Scales of rows of whole 16 bytes that start between them."""
    assert cl.lib().cascadia_int4_debug_fp8_gemm_form(n, k, 2, m, 0) == form
    w, ws, x, xs = (t.cuda() for t in gemm_case(m, m, n, k, "fp8"))
    ys = []
    for at in (0, 1):
        wide = torch.empty(xs.numel() + 1, device="cuda")
        wide[at:at + xs.numel()] = xs.view(-1)
        ww = torch.empty(ws.numel() + 1, device="cuda")
        ww[at:at + ws.numel()] = ws.view(-1)
        y = torch.empty((m, n), dtype=BF16, device="cuda")
        cl.fp8_gemm(w, ww[at:at + ws.numel()], x, n, k, m, y, x_scales=wide[at:at + xs.numel()])
        ys.append(y)
    assert torch.equal(*ys)


@pytest.mark.parametrize("out_dtype", [F32, BF16])
def test_one_token_slots_left_out(cl, out_dtype):
    g = gen(23)
    for ids in ([[-1, 2, 7, 2 ** 31 - 1]], [[1, 1, 1, 1]], [[-5, -1, 6, 9]], [[3, 2, 1, 0]]):
        case = moe_case(3, 1, 272, 144, 6, 4, BF16, torch.tensor(ids))
        case[6][0, 3] = 0.05
        check_moe(cl, case, out_dtype, threshold=0.1)
        check_moe(cl, case, out_dtype, threshold=0.1, residual=False)
    res = case[-1].to(out_dtype)
    out = run_moe(cl, case, out_dtype, 2.0, res)  # every weight below the threshold
    assert torch.equal(out.cpu(), res)


@pytest.mark.parametrize("T,H,I,E,k", [(1, 16400, 16, 3, 2), (5, 16400, 16, 8, 2), (9, 16400, 48, 2, 2),
                                       (1, 48, 16400, 2, 1), (3, 16, 16400, 6, 2)])
def test_very_wide_layers(cl, T, H, I, E, k):
    for dt in (F32, BF16):
        check_moe(cl, moe_case(T + H, T, H, I, E, k, BF16), dt)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("norm", [True, False])
def test_route_weights_round_once(cl, score, norm):
    """Scores, their sum, the division and the scale in 64 bits and one rounding at the
    end.  (A softmax's sum adds exponentials e of 32 bits: each off by 2^-23 of itself,
    and by half a step of its argument d, which renormalising takes out of the weights.)"""
    logits = normal(gen(24), 300, 256) * 2
    _, w = run_route(cl, logits, 8, score, None, 1, 1, 1, norm, 2.5)
    _, want = ref.route(logits.double().numpy(), 8, score, None, 1, 1, 1, norm, 2.5)
    steps = np.ones((300, 1))
    if score == "softmax" and not norm:
        d = (logits.max(1, keepdim=True).values - logits).double().numpy()
        steps += (np.exp(-d) * (2 + d)).sum(1, keepdims=True) / np.exp(-d).sum(1, keepdims=True)
    assert np.all(np.abs(w - want) <= steps * (1 + 1e-6) * ref.U32 * np.abs(want))
