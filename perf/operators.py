"""Performance cases of expert routing and of the 8-bit floating-point products.

Four operators of the serving path, each through its public entry point of
`cascadia_amd`, beside its plain form in elementary torch operations:

  route     choice of a layer's experts from its router logits: softmax or
            sigmoid scores, a bias for balance, groups, top-k, renormalised
  quantize  e4m3 codes and f32 scales of activations (groups of 128 along a
            row) and of weights (blocks of 128 x 128, at load)
  gemm      product of e4m3 matrices with a scale per block of 128
  moe       a layer's experts in e4m3: gate / up, SwiGLU, requantised, down,
            the weighted sum of the chosen experts

Every input is made from the seed alone.  Weights are normal values held in
e4m3 with the scale of a block whose largest value is four deviations, so that
products have unit size; activations N(0, 1) with a few wide channels; router
logits N(0, 1.5) per expert, even or with a Zipf skew.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BLOCK = 128
E4M3_MAX = 448.0
LEAST = 2.0 ** -96  # the least absolute maximum of a group
FP8 = torch.float8_e4m3fn
ZIPF = 1.1
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "fp8": FP8}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one decoded token's choice among 256 experts in 8 groups (latency)
        _route("route_one_token", tokens=1, experts=256, top_k=8, score="sigmoid", bias=True,
               groups=8, top_groups=4, best=2, norm=True, scale=2.5, x="f32"),
        # a prompt's choice by softmax from bf16 logits, an odd number of
        # experts, weights as the softmax gives them
        _route("route_softmax_bf16_333", tokens=333, experts=60, top_k=4, score="softmax",
               bias=False, groups=1, top_groups=1, best=1, norm=False, scale=1.0, x="bf16"),
        # a large prefill batch over 384 experts, balanced by a bias
        _route("route_prefill_8192", tokens=8192, experts=384, top_k=8, score="sigmoid", bias=True,
               groups=1, top_groups=1, best=1, norm=True, scale=2.5, x="f32"),
        # a prompt's activations on the way into a product
        _quant("quantize_rows_4096", rows=4096, cols=7168, x="bf16", blocks=False),
        # loading: a matrix of the model shell, ragged in both directions
        _quant("quantize_blocks_7104", rows=7104, cols=8112, x="bf16", blocks=True),
        # the smallest product: one decoded token, its row quantised in the call
        _gemm("gemm_one_token", rows=1, n=4096, k=4096, x="bf16", y="bf16"),
        # a decode batch over an FFN's width
        _gemm("gemm_batch_16", rows=16, n=14336, k=4096, x="bf16", y="bf16"),
        # a ragged prompt over a narrow projection (4.5 blocks), codes in hand
        _gemm("gemm_ragged_333", rows=333, n=576, k=7168, x="fp8", y="f32"),
        # a long prompt over an FFN's width
        _gemm("gemm_prefill_4096", rows=4096, n=14336, k=4096, x="fp8", y="bf16"),
        # a layer of 384 experts: one decoded token
        _moe("moe_384_one_token", tokens=1, hidden=7168, inter=2048, experts=384, top_k=8,
             skew="even", x="bf16"),
        # a decode batch over 60 experts, f32 activations as that runner holds them
        _moe("moe_60_batch_32", tokens=32, hidden=3584, inter=1408, experts=60, top_k=8,
             skew="zipf", x="f32"),
        # a prompt over 128 experts
        _moe("moe_128_prefill_2048", tokens=2048, hidden=4096, inter=1536, experts=128, top_k=8,
             skew="zipf", x="bf16"),
    ]


def _route(name, tokens, experts, top_k, score, bias, groups, top_groups, best, norm, scale, x):
    return {"name": name, "kind": "route", "tokens": tokens, "experts": experts, "top_k": top_k,
            "score": score, "bias": bias, "groups": groups, "top_groups": top_groups,
            "best": best, "norm": norm, "scale": scale, "x": x}


def _quant(name, rows, cols, x, blocks):
    return {"name": name, "kind": "quantize", "rows": rows, "cols": cols, "x": x, "blocks": blocks}


def _gemm(name, rows, n, k, x, y):
    return {"name": name, "kind": "gemm", "rows": rows, "n": n, "k": k, "x": x, "y": y}


def _moe(name, tokens, hidden, inter, experts, top_k, skew, x):
    return {"name": name, "kind": "moe", "tokens": tokens, "hidden": hidden, "inter": inter,
            "experts": experts, "top_k": top_k, "skew": skew, "x": x}


def _log(rng, lo, hi):
    """An integer of [lo, hi], its logarithm uniform."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["route", "quantize", "gemm", "gemm", "moe", "moe"])
    if kind == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * _log(rng, 16, 480 // groups) if groups > 1 else _log(rng, 16, 480)
        top_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(8, top_groups * (experts // groups)))
        c = _route("", _log(rng, 1, 8192), experts, top_k, rng.choice(["softmax", "sigmoid"]),
                   rng.choice([True, False]), groups, top_groups, rng.choice([1, 2]),
                   rng.choice([True, False]), rng.choice([1.0, 2.5]), rng.choice(["f32", "bf16"]))
        while c["tokens"] * c["experts"] > 8192 * 384:
            c["tokens"] = (c["tokens"] + 1) // 2
    elif kind == "quantize":
        blocks = rng.choice([True, False])
        c = _quant("", _log(rng, 1, 8192), 16 * _log(rng, 8, 896),
                   "bf16" if blocks else rng.choice(["bf16", "f32"]), blocks)
        while c["rows"] * c["cols"] > 7104 * 8112 // (2 if c["x"] == "f32" else 1):
            c["rows"] = (c["rows"] + 1) // 2
    elif kind == "gemm":
        c = _gemm("", _log(rng, 1, 4096), _log(rng, 256, 14336), 16 * _log(rng, 16, 896),
                  rng.choice(["bf16", "f32", "fp8", "fp8"]), rng.choice(["bf16", "f32"]))
        while c["rows"] * c["n"] * c["k"] > 4096 * 14336 * 4096:
            c["rows"] = (c["rows"] + 1) // 2
    else:
        c = _moe("", _log(rng, 1, 2048), 64 * _log(rng, 16, 112), 32 * _log(rng, 16, 64),
                 rng.choice([16, 60, 128, 256]), rng.randint(2, 8), rng.choice(["even", "zipf"]),
                 rng.choice(["bf16", "f32"]))
        while c["experts"] * c["hidden"] * c["inter"] > 128 * 4096 * 1536:
            c["experts"] = c["experts"] * 3 // 4
        c["experts"] = max(10, c["experts"])
        while c["tokens"] * c["top_k"] * c["hidden"] * c["inter"] > 2048 * 8 * 4096 * 1536:
            c["tokens"] = (c["tokens"] + 1) // 2
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------

def _gen(seed, device=DEV):
    g = torch.Generator(device=device)
    g.manual_seed(int(seed) * 7919 + 101)
    return g


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _codes(g, shape):
    """e4m3 values of a block whose largest is about four deviations."""
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)
    return x.mul_(E4M3_MAX / 4).clamp_(-E4M3_MAX, E4M3_MAX).to(FP8)


def _weight_scales(g, *shape, k):
    """Scales that give the weights a deviation of about 1 / sqrt(k)."""
    s = torch.rand(shape, generator=g, device=DEV).add_(0.5)
    return s.mul_(4 / (E4M3_MAX * math.sqrt(k)))


def _weight(g, n, k):
    return _codes(g, (n, k)), _weight_scales(g, _blocks(n), _blocks(k), k=k)


def _act(g, rows, cols, kind):
    x = torch.randn((rows, cols), generator=g, device=DEV)
    wide = torch.rand(cols, generator=g, device=DEV) < 0.005
    x = torch.where(wide[None, :], x * 8, x)
    return x if kind == "f32" else x.to(torch.bfloat16)


def _logits(case, g, device):
    v = torch.randn((case["tokens"], case["experts"]), generator=g, device=device) * 1.5
    if case.get("skew") == "zipf":
        order = torch.randperm(case["experts"], generator=g, device=device)
        v -= ZIPF * torch.log1p(order.float())[None, :]
    return v


def _moe_routing(case, seed):
    """ids and weights of a layer's tokens: the chosen logits' softmax."""
    v, ids = torch.topk(_logits(case, _gen(seed, "cpu"), "cpu"), case["top_k"], dim=1)
    return ids.to(torch.int32).to(DEV), torch.softmax(v, dim=1).to(DEV)


def _route_inputs(case, seed):
    g = _gen(seed)
    logits = _logits(case, g, DEV).to(DTYPES[case["x"]])
    bias = torch.randn(case["experts"], generator=g, device=DEV).mul_(0.05) if case["bias"] else None
    return logits, bias


def _quant_inputs(case, seed):
    g = _gen(seed)
    if case["blocks"]:
        w = torch.randn((case["rows"], case["cols"]), generator=g, device=DEV).mul_(0.02)
        return w.to(torch.bfloat16)
    return _act(g, case["rows"], case["cols"], case["x"])


def _gemm_inputs(case, seed):
    g = _gen(seed)
    w, ws = _weight(g, case["n"], case["k"])
    if case["x"] == "fp8":
        x = _codes(g, (case["rows"], case["k"]))
        xs = torch.rand((case["rows"], _blocks(case["k"])), generator=g, device=DEV)
        return w, ws, x, xs.add_(0.5).mul_(4 / E4M3_MAX)
    return w, ws, _act(g, case["rows"], case["k"], case["x"]), None


def _moe_inputs(case, seed):
    g = _gen(seed)
    e, h, i = case["experts"], case["hidden"], case["inter"]
    gate_up = torch.empty((e, 2, i, h), device=DEV, dtype=FP8)
    down = torch.empty((e, h, i), device=DEV, dtype=FP8)
    for j in range(e):
        gate_up[j] = _codes(g, (2, i, h))
        down[j] = _codes(g, (h, i))
    gate_up_s = _weight_scales(g, e, 2, _blocks(i), _blocks(h), k=h)
    down_s = _weight_scales(g, e, _blocks(h), _blocks(i), k=i)
    x = _act(g, case["tokens"], h, case["x"])
    residual = torch.randn((case["tokens"], h), generator=g, device=DEV).to(torch.bfloat16)
    return gate_up, gate_up_s, down, down_s, x, residual


# ---------------------------------------------------------------------------
# prepare / run
# ---------------------------------------------------------------------------

def prepare(case, seed):
    return {"route": _prepare_route, "quantize": _prepare_quant, "gemm": _prepare_gemm,
            "moe": _prepare_moe}[case["kind"]](case, seed)


def run(state):
    return state["run"](state)


def _prepare_route(case, seed):
    logits, bias = _route_inputs(case, seed)
    shape = (case["tokens"], case["top_k"])
    st = {"run": _run_route, "case": case, "logits": logits, "bias": bias,
          "ids": torch.empty(shape, dtype=torch.int32, device=DEV),
          "weights": torch.empty(shape, dtype=torch.float32, device=DEV)}
    if own:
        import cascadia_amd as cl
        st["score"] = cl.SCORE_SOFTMAX if case["score"] == "softmax" else cl.SCORE_SIGMOID
    return st


def _run_route(st):
    c = st["case"]
    if own:
        import cascadia_amd as cl
        cl.route_experts(st["logits"], c["top_k"], st["ids"], st["weights"], score=st["score"],
                         bias=st["bias"], n_groups=c["groups"], top_groups=c["top_groups"],
                         group_best=c["best"], normalize=c["norm"], scale=c["scale"])
        return {"ids": st["ids"], "weights": st["weights"]}
    ids, w = _plain_route(c, st["logits"], st["bias"])
    return {"ids": ids.to(torch.int32), "weights": w}


def _first(keys, count):
    """Places of the `count` largest keys of each row, ties to the lower place."""
    return torch.sort(keys, dim=-1, descending=True, stable=True).indices[..., :count]


def _plain_route(c, logits, bias):
    # (64 bits: two experts' scores may lie closer than 32 bits tell apart)
    v = logits.double()
    if c["score"] == "softmax":
        s = torch.exp(v - v.amax(1, keepdim=True))
        s = s / s.sum(1, keepdim=True)
    else:
        s = 1.0 / (1.0 + torch.exp(-v))
    key = s + bias.double() if bias is not None else s
    order = key if bias is not None else v
    if c["groups"] > 1:
        t, e, gr = c["tokens"], c["experts"], c["groups"]
        best = torch.sort(key.view(t, gr, e // gr), dim=2, descending=True).values
        kept = _first(best[:, :, :c["best"]].sum(2), c["top_groups"])
        keep = torch.zeros((t, gr), dtype=torch.bool, device=v.device).scatter_(1, kept, True)
        order = torch.where(keep.repeat_interleave(e // gr, 1), order,
                            torch.full_like(order, -math.inf))
    ids = _first(order, c["top_k"])
    w = s.gather(1, ids)
    if c["norm"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return ids, (w * c["scale"]).float()


def _prepare_quant(case, seed):
    x = _quant_inputs(case, seed)
    st = {"run": _run_quant, "case": case, "x": x}
    if not case["blocks"]:
        st["codes"] = torch.empty(x.shape, dtype=FP8, device=DEV)
        st["scales"] = torch.empty((case["rows"], _blocks(case["cols"])), dtype=torch.float32,
                                   device=DEV)
    return st


def _run_quant(st):
    c = st["case"]
    if own:
        import cascadia_amd as cl
        if c["blocks"]:
            codes, scales = cl.quantize_fp8_blocks(st["x"], c["rows"], c["cols"])
        else:
            codes, scales = cl.quantize_fp8(st["x"], c["rows"], c["cols"], st["codes"],
                                            st["scales"])
        return {"codes": codes, "scales": scales}
    codes, scales = _plain_blocks(st["x"]) if c["blocks"] else _plain_rows(st["x"])
    return {"codes": codes, "scales": scales}


def _divided(f, top):
    """f (grouped, with its groups' maxima top) as e4m3 codes, and their scales.
    (64 bits, and the quotient itself: bf16 values often lie halfway between two
    codes, where a rounded 448 / top would choose by chance)"""
    top = top.double()
    q = f.double() * E4M3_MAX / top
    return q.float().to(FP8), (top / E4M3_MAX).float()


def _plain_rows(x):
    """e4m3 codes [rows, cols] and scales [rows, blocks] of groups of 128."""
    rows, cols = x.shape
    kb = _blocks(cols)
    f = torch.nn.functional.pad(x.float(), (0, kb * BLOCK - cols)).view(rows, kb, BLOCK)
    q, scales = _divided(f, f.abs().amax(2, keepdim=True).clamp(min=LEAST))
    return q.view(rows, kb * BLOCK)[:, :cols].contiguous(), scales.view(rows, kb)


def _plain_blocks(w):
    """e4m3 codes [rows, cols] and scales of blocks of 128 x 128."""
    rows, cols = w.shape
    nb, kb = _blocks(rows), _blocks(cols)
    f = torch.nn.functional.pad(w.float(), (0, kb * BLOCK - cols, 0, nb * BLOCK - rows))
    f = f.view(nb, BLOCK, kb, BLOCK)
    q, scales = _divided(f, f.abs().amax((1, 3), keepdim=True).clamp(min=LEAST))
    return q.view(nb * BLOCK, kb * BLOCK)[:rows, :cols].contiguous(), scales.view(nb, kb)


def _spread(s, n, k):
    """Scales of blocks [..., blocks of n, blocks of k] over their values."""
    s = s.repeat_interleave(BLOCK, -2)[..., :n, :]
    return s.repeat_interleave(BLOCK, -1)[..., :k]


def _prepare_gemm(case, seed):
    w, ws, x, xs = _gemm_inputs(case, seed)
    st = {"run": _run_gemm, "case": case, "w": w, "ws": ws, "x": x, "xs": xs, "ws_buf": None,
          "y": torch.empty((case["rows"], case["n"]), dtype=DTYPES[case["y"]], device=DEV)}
    if own:
        import cascadia_amd as cl
        need = cl.fp8_gemm_workspace_bytes(case["n"], case["k"], case["rows"], x.dtype)
        st["ws_buf"] = torch.empty(max(256, need), dtype=torch.uint8, device=DEV)
    return st


def _run_gemm(st):
    c = st["case"]
    if own:
        import cascadia_amd as cl
        return cl.fp8_gemm(st["w"], st["ws"], st["x"], c["n"], c["k"], c["rows"], st["y"],
                           x_scales=st["xs"], workspace=st["ws_buf"])
    x, xs = (st["x"], st["xs"]) if st["xs"] is not None else _plain_rows(st["x"])
    xd = x.float() * xs.repeat_interleave(BLOCK, 1)[:, :c["k"]]
    wd = st["w"].float() * _spread(st["ws"], c["n"], c["k"])
    return (xd @ wd.T).to(DTYPES[c["y"]])


def _prepare_moe(case, seed):
    gate_up, gate_up_s, down, down_s, x, residual = _moe_inputs(case, seed)
    ids, weights = _moe_routing(case, seed)
    st = {"run": _run_moe, "case": case, "gate_up": gate_up, "gate_up_s": gate_up_s, "down": down,
          "down_s": down_s, "x": x, "residual": residual, "ids": ids, "weights": weights,
          "out": torch.empty_like(residual)}
    if own:
        import cascadia_amd as cl
        st["experts"] = cl.Fp8Experts(gate_up, gate_up_s, down, down_s, case["experts"],
                                      case["hidden"], case["inter"])
        need = cl.fp8_moe_workspace_bytes(st["experts"], case["top_k"], case["tokens"])
        st["ws_buf"] = torch.empty(need, dtype=torch.uint8, device=DEV)
    return st


def _run_moe(st):
    c = st["case"]
    if own:
        import cascadia_amd as cl
        return cl.fp8_moe_forward(st["experts"], st["x"], st["out"], top_k=c["top_k"],
                                  ids=st["ids"], weights=st["weights"], residual=st["residual"],
                                  workspace=st["ws_buf"])
    t, k, h, i = c["tokens"], c["top_k"], c["hidden"], c["inter"]
    xq, xs = _plain_rows(st["x"])
    xd = xq.float() * xs.repeat_interleave(BLOCK, 1)[:, :h]
    # the chosen experts' rows side by side, padded to the longest
    active, at = torch.unique(st["ids"].flatten().long(), return_inverse=True)
    order = torch.argsort(at, stable=True)
    count = torch.bincount(at)
    start = torch.cumsum(count, 0) - count
    place = torch.empty_like(at)
    place[order] = torch.arange(t * k, device=at.device) - start[at[order]]
    rows = torch.zeros((active.numel(), int(count.max()), h), device=at.device)
    rows[at, place] = xd.repeat_interleave(k, 0)
    gate, up = (rows @ (st["gate_up"][active, j].float()
                        * _spread(st["gate_up_s"][active, j], i, h)).transpose(1, 2)
                for j in (0, 1))
    mid = gate / (1 + torch.exp(-gate)) * up
    mq, ms = _plain_rows(mid.view(-1, i))
    mid = (mq.float() * ms.repeat_interleave(BLOCK, 1)[:, :i]).view(mid.shape)
    y = mid @ (st["down"][active].float() * _spread(st["down_s"][active], h, i)).transpose(1, 2)
    y = y[at, place].view(t, k, h) * st["weights"].unsqueeze(2)
    return (st["residual"].float() + y.sum(1)).to(torch.bfloat16)


# ---------------------------------------------------------------------------
# what one pass cannot do without
# ---------------------------------------------------------------------------

def _bytes_of(kind):
    return {"f32": 4, "bf16": 2, "fp8": 1}[kind]


def work(case):
    if case["kind"] == "route":
        n = case["tokens"] * case["experts"]
        return {"bytes": n * _bytes_of(case["x"]) + case["tokens"] * case["top_k"] * 8
                + (case["experts"] * 4 if case["bias"] else 0), "flops": 25 * n}
    if case["kind"] == "quantize":
        r, k = case["rows"], case["cols"]
        scales = (_blocks(r) if case["blocks"] else r) * _blocks(k) * 4
        return {"bytes": r * k * (_bytes_of(case["x"]) + 1) + scales, "flops": 4 * r * k}
    if case["kind"] == "gemm":
        m, n, k = case["rows"], case["n"], case["k"]
        b = n * k + _blocks(n) * _blocks(k) * 4 + m * n * _bytes_of(case["y"])
        b += m * k * _bytes_of(case["x"]) + (m * _blocks(k) * 4 if case["x"] == "fp8" else 0)
        return {"bytes": b, "flops": 2 * m * n * k}
    t, h, i, k = case["tokens"], case["hidden"], case["inter"], case["top_k"]
    active = sum(torch.topk(_logits(case, _gen(s, "cpu"), "cpu"), k, dim=1).indices.unique().numel()
                 for s in range(4)) / 4
    per = 3 * h * i + 3 * _blocks(h) * _blocks(i) * 4
    return {"bytes": active * per + t * h * (_bytes_of(case["x"]) + 4) + t * k * 8,
            "flops": 6 * t * k * h * i}


# ---------------------------------------------------------------------------
# what a pass returns, in 64 bits
# ---------------------------------------------------------------------------

def _e4m3_64(v):
    """v rounded to e4m3 (3 mantissa bits, least exponent -6), to nearest even."""
    e = torch.frexp(v).exponent.clamp(min=-5)  # v = m 2^e with 0.5 <= m < 1
    step = torch.ldexp(torch.ones_like(v), e - 4)
    return torch.round(v / step) * step


def _rows64(x):
    """x (float64 [rows, cols]) as its e4m3 codes and scales stand for it."""
    rows, cols = x.shape
    out = torch.empty_like(x)
    scales = torch.empty((rows, _blocks(cols)), dtype=torch.float64, device=x.device)
    for b in range(_blocks(cols)):
        part = x[:, b * BLOCK:(b + 1) * BLOCK]
        top = part.abs().max(1, keepdim=True).values.clamp(min=LEAST)
        out[:, b * BLOCK:(b + 1) * BLOCK] = _e4m3_64(part * E4M3_MAX / top)
        scales[:, b:b + 1] = top / E4M3_MAX
    return out, scales


def _value64(codes, scales, row_block):
    """Codes [n, k] times their blocks' scales, in 64 bits."""
    n, k = codes.shape
    out = codes.double()
    r = torch.arange(n, device=out.device) // row_block
    c = torch.arange(k, device=out.device) // BLOCK
    return out.mul_(scales.double()[r][:, c])


def exact(case, seed):
    if case["kind"] == "route":
        return _exact_route(case, seed)
    if case["kind"] == "quantize":
        return _exact_quant(case, seed)
    if case["kind"] == "gemm":
        w, ws, x, xs = _gemm_inputs(case, seed)
        x, xs = _rows64(x.double()) if xs is None else (x, xs)
        return _value64(x, xs, 1) @ _value64(w, ws, BLOCK).T
    return _exact_moe(case, seed)


def _exact_route(case, seed):
    logits, bias = _route_inputs(case, seed)
    s = logits.double()
    s = torch.sigmoid(s) if case["score"] == "sigmoid" else torch.softmax(s, 1)
    c = s if bias is None else s + bias.double()
    per = case["experts"] // case["groups"]
    if case["groups"] > 1:
        g = torch.topk(c.view(-1, case["groups"], per), min(case["best"], per), dim=2).values.sum(2)
        left = torch.zeros_like(g, dtype=torch.bool)
        left.scatter_(1, torch.topk(g, case["top_groups"], dim=1).indices, True)
        c = c.masked_fill(~left.repeat_interleave(per, 1), -math.inf)
    w = s.gather(1, torch.topk(c, case["top_k"], dim=1).indices)
    if case["norm"]:
        w = w / w.sum(1, keepdim=True)
    return {"ids": None, "weights": w * case["scale"]}


def _exact_quant(case, seed):
    x = _quant_inputs(case, seed).double()
    if not case["blocks"]:
        codes, scales = _rows64(x)
        return {"codes": codes, "scales": scales}
    codes = torch.empty_like(x)
    scales = torch.empty((_blocks(x.shape[0]), _blocks(x.shape[1])), dtype=torch.float64,
                         device=x.device)
    for r in range(scales.shape[0]):
        band = x[r * BLOCK:(r + 1) * BLOCK]
        top = band.abs().max(0).values
        top = torch.nn.functional.pad(top, (0, scales.shape[1] * BLOCK - x.shape[1]))
        top = top.view(-1, BLOCK).max(1).values.clamp(min=LEAST)
        scales[r] = top / E4M3_MAX
        each = top.repeat_interleave(BLOCK)[:x.shape[1]]
        codes[r * BLOCK:(r + 1) * BLOCK] = _e4m3_64(band * E4M3_MAX / each[None, :])
    return {"codes": codes, "scales": scales}


def _exact_moe(case, seed):
    gate_up, gate_up_s, down, down_s, x, residual = _moe_inputs(case, seed)
    ids, weights = _moe_routing(case, seed)
    xd = _value64(*_rows64(x.double()), 1)
    out = residual.double()
    for e in ids.unique().tolist():
        tok, slot = (ids == e).nonzero(as_tuple=True)
        g, u = (xd[tok] @ _value64(gate_up[e, j], gate_up_s[e, j], BLOCK).T for j in (0, 1))
        mid = _value64(*_rows64(g * torch.sigmoid(g) * u), 1)
        y = mid @ _value64(down[e], down_s[e], BLOCK).T
        out.index_add_(0, tok, y * weights.double()[tok, slot].unsqueeze(1))
    return out
