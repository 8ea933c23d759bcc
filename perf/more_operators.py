"""Performance cases of tokens sorted by expert and back, and of low-rank adapters.

Operators of a sparse-MoE layer whose experts are run one by one (or on another
rank), and of a projection that many requests share, each through its public
entry point of `cascadia_amd`, beside its plain form in elementary torch
operations:

  sort      slots of chosen experts -> rows in order of their expert (stable),
            and back; the same call groups a batch's rows by adapter
  gather    a token's row to each of its slots' rows
  combine   the weighted sum of a token's slots and a residual; without weights
            it is the gradient of gather
  grad      the gradient of combine: of the slots' rows and of the weights
  adapters  ys = base + s B_a (A_a x), a row's own adapter a: the rows of many
            requests at once beside a projection that they share

Every input is made from the seed alone.  Router logits N(0, 1.5) per expert,
even or with a Zipf skew; the last tokens of a padded batch have no expert (ids
-1).  Activations N(0, 1) with a few wide channels; an adapter's inner values
have unit size, and its output is a tenth or so of the projection's.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
ZIPF = 1.1
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # a decode batch of 16 over 256 experts (latency)
        _sort("sort_batch_16", tokens=16, top_k=8, experts=256, skew="even", padded=0, weights=False),
        # a padded prefill batch over 384 experts, slots of small weight left out
        _sort("sort_prefill_8192", tokens=8192, top_k=8, experts=384, skew="zipf", padded=237,
              weights=True),
        # a decode batch over 60 experts, f32 activations to the experts' bf16
        _move("gather_batch_32", "gather", tokens=32, top_k=8, experts=60, hidden=3584, skew="zipf",
              padded=0, x="f32", y="bf16"),
        # a padded prompt's rows
        _move("gather_prefill_4096", "gather", tokens=4096, top_k=8, experts=384, hidden=7168,
              skew="zipf", padded=113, x="bf16", y="bf16"),
        # an odd number of tokens, f32 rows into the bf16 stream
        _move("combine_333", "combine", tokens=333, top_k=4, experts=60, hidden=4096, skew="zipf",
              padded=5, x="f32", y="bf16"),
        # a padded prompt's slots
        _move("combine_prefill_4096", "combine", tokens=4096, top_k=8, experts=384, hidden=7168,
              skew="zipf", padded=113, x="bf16", y="bf16"),
        # the gradient of gather in a training step
        _move("gather_grad_2048", "spread", tokens=2048, top_k=6, experts=128, hidden=4096,
              skew="even", padded=0, x="bf16", y="f32"),
        # a short ragged sequence's gradient in f32
        _move("grad_77", "grad", tokens=77, top_k=6, experts=60, hidden=3584, skew="even", padded=3,
              x="f32", y="f32"),
        # a training step over a padded batch
        _move("grad_4096", "grad", tokens=4096, top_k=8, experts=128, hidden=4096, skew="zipf",
              padded=113, x="bf16", y="bf16"),
        # one decoded token beside an attention-sized projection (latency)
        _adapt("adapters_one_token", tokens=1, requests=1, adapters=16, bare=0.0, rank=16, mixed=False,
               k=4096, n=4096, x="bf16", base="bf16", y="bf16"),
        # a decode batch of many requests, mixed ranks, some without an adapter
        _adapt("adapters_batch_64", tokens=64, requests=64, adapters=100, bare=0.2, rank=64, mixed=True,
               k=4096, n=14336, x="f32", base="f32", y="f32"),
        # prompts of nine requests
        _adapt("adapters_prefill_4096", tokens=4096, requests=9, adapters=16, bare=0.2, rank=32,
               mixed=False, k=4096, n=14336, x="bf16", base="bf16", y="bf16"),
    ]


def _sort(name, tokens, top_k, experts, skew, padded, weights):
    return {"name": name, "kind": "sort", "tokens": tokens, "top_k": top_k, "experts": experts,
            "skew": skew, "padded": padded, "weights": weights}


def _move(name, kind, tokens, top_k, experts, hidden, skew, padded, x, y):
    """x: the type read per slot (gather: per token), y: the other side's."""
    return {"name": name, "kind": kind, "tokens": tokens, "top_k": top_k, "experts": experts,
            "hidden": hidden, "skew": skew, "padded": padded, "x": x, "y": y}


def _adapt(name, tokens, requests, adapters, bare, rank, mixed, k, n, x, base, y):
    """base: the projection's output type, or "none"; bare: the share of requests
    without an adapter; mixed: ranks of 4 up to `rank`, else all of `rank`."""
    return {"name": name, "kind": "adapters", "tokens": tokens, "requests": requests,
            "adapters": adapters, "bare": bare, "rank": rank, "mixed": mixed, "k": k, "n": n,
            "x": x, "base": base, "y": y}


def _log(rng, lo, hi):
    """An integer of [lo, hi], its logarithm uniform."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


MOST_SLOT_VALUES = 4096 * 8 * 7168   # rows of the largest gather, combine
MOST_GRAD_VALUES = 4096 * 8 * 4096
MOST_ADAPTED = 4096 * (4096 + 2 * 14336)
MOST_ADAPTERS = 1 << 28              # values of all A and B


def draw(rng):
    kind = rng.choice(["sort", "gather", "combine", "spread", "grad", "adapters", "adapters",
                       "adapters"])
    skew, f = rng.choice(["even", "zipf"]), ["f32", "bf16"]
    if kind == "adapters":
        tokens = _log(rng, 1, 4096)
        c = _adapt("", tokens, _log(rng, 1, min(tokens, 256)), _log(rng, 1, 256),
                   rng.choice([0.0, 0.2]), 8 * rng.choice([1, 1, 2, 2, 3, 4, 5, 8, 8, 16]),
                   rng.choice([True, False]), 8 * _log(rng, 128, 1792), _log(rng, 256, 14336),
                   rng.choice(f), rng.choice(f + ["none"]), rng.choice(f))
        while c["adapters"] * c["rank"] * (c["k"] + c["n"]) > MOST_ADAPTERS:
            c["adapters"] = c["adapters"] * 3 // 4
        wide = _bytes_of(c["x"]) * c["k"] + (_bytes_of(c["base"]) + _bytes_of(c["y"])) * c["n"]
        while c["tokens"] * wide > 2 * MOST_ADAPTED:
            c["tokens"] = (c["tokens"] + 1) // 2
        c["requests"] = min(c["requests"], c["tokens"])
    else:
        experts = _log(rng, 8, 512)
        tokens, top_k = _log(rng, 1, 8192), rng.randint(1, 8)
        padded = rng.choice([0, rng.randint(0, tokens // 16)])
        if kind == "sort":
            c = _sort("", tokens, top_k, experts, skew, padded, rng.choice([True, False]))
        else:
            hidden = 8 * _log(rng, 64, 896) if rng.random() < 0.75 else _log(rng, 512, 7168)
            c = _move("", kind, tokens, top_k, experts, hidden, skew, padded, rng.choice(f),
                      rng.choice(f))
            most = MOST_GRAD_VALUES if kind == "grad" else MOST_SLOT_VALUES
            per = top_k * c["hidden"] * (_bytes_of(c["x"]) + _bytes_of(c["y"])) / 4
            while c["tokens"] * per > most:
                c["tokens"] = (c["tokens"] + 1) // 2
            c["padded"] = min(padded, c["tokens"] // 16)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------

def _gen(seed, device=None):
    g = torch.Generator(device=device or DEV)
    g.manual_seed(int(seed) * 7919 + 211)
    return g


def _bytes_of(kind):
    return {"f32": 4, "bf16": 2, "none": 0}[kind]


def _act(g, rows, cols, kind):
    x = torch.randn((rows, cols), generator=g, device=DEV)
    wide = torch.rand(cols, generator=g, device=DEV) < 0.005
    return torch.where(wide[None, :], x * 8, x).to(DTYPES[kind])


def _zipf(case, experts, g):
    """Log odds of each expert (CPU)."""
    v = torch.zeros(experts)
    if case.get("skew") == "zipf":
        v -= ZIPF * torch.log1p(torch.randperm(experts, generator=g).float())
    return v


def _routing(case, seed):
    """ids and weights of a batch's slots (CPU): the chosen logits' softmax."""
    g = _gen(seed, "cpu")
    odds = _zipf(case, case["experts"], g)
    logits = torch.randn((case["tokens"], case["experts"]), generator=g) * 1.5 + odds
    v, ids = torch.topk(logits, min(case["top_k"], case["experts"]), dim=1)
    ids = ids.to(torch.int32)
    if case["padded"]:
        ids[-case["padded"]:] = -1
    return ids, torch.softmax(v, dim=1)


THRESHOLD = 2.0 ** -6  # slots of less weight are left out, where a case has weights


def _kept(case, ids, weights):
    in_ = (ids >= 0) & (ids < case["experts"])
    return in_ & ~(weights < THRESHOLD) if case.get("weights") else in_


def _plain_sort(ids, kept, experts):
    """offsets, slots, rows from their definition (any device)."""
    n = ids.numel()
    key = torch.where(kept, ids, torch.full_like(ids, experts)).view(-1)
    slots = torch.sort(key, stable=True).indices
    count = torch.bincount(key, minlength=experts + 1)[:experts]
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device)
    offsets[1:] = torch.cumsum(count, 0)
    rows = torch.empty(n, dtype=torch.int64, device=ids.device)
    rows[slots] = torch.arange(n, device=ids.device)
    rows = torch.where(kept.view(-1), rows, torch.full_like(rows, -1))
    return offsets.int(), slots.int(), rows.int().view(ids.shape)


def _sort_inputs(case, seed):
    ids, weights = _routing(case, seed)
    return ids.to(DEV), weights.to(DEV)


def _move_inputs(case, seed):
    ids, weights = _routing(case, seed)
    rows = _plain_sort(ids, _kept(case, ids, weights), case["experts"])[2].to(DEV)
    g = _gen(seed)
    n, h = case["tokens"] * case["top_k"], case["hidden"]
    t = {"rows": rows, "weights": weights.to(DEV)}
    if case["kind"] == "gather":
        t["x"] = _act(g, case["tokens"], h, case["x"])
        return t
    t["ys"] = torch.randn((n, h), generator=g, device=DEV, dtype=DTYPES[case["x"]])
    if case["kind"] == "combine":
        t["residual"] = _act(g, case["tokens"], h, case["y"])
    if case["kind"] == "grad":
        t["dout"] = torch.randn((case["tokens"], h), generator=g, device=DEV).to(DTYPES[case["y"]])
    return t


def _requests(case, seed):
    """Adapter of each row (CPU): contiguous rows of a request share one."""
    g = _gen(seed, "cpu")
    t, r = case["tokens"], case["requests"]
    cuts = torch.randperm(t - 1, generator=g)[:r - 1] + 1 if r > 1 else torch.empty(0, dtype=torch.long)
    first = torch.zeros(t, dtype=torch.long)
    first[cuts] = 1
    odds = torch.softmax(-torch.log1p(torch.arange(case["adapters"]).float()), 0)
    pick = torch.multinomial(odds, r, replacement=True, generator=g)
    bare = torch.rand(r, generator=g) < case["bare"]
    bare[0] = False
    pick[bare] = -1
    return pick[torch.cumsum(first, 0)].to(torch.int32)


def _ranks(case, seed):
    g = _gen(seed + 1, "cpu")
    if not case["mixed"]:
        return [case["rank"]] * case["adapters"]
    return torch.randint(4, case["rank"] + 1, (case["adapters"],), generator=g).tolist()


def _adapt_inputs(case, seed):
    g = _gen(seed)
    e, r, k, n = case["adapters"], case["rank"], case["k"], case["n"]
    a = torch.randn((e, r, k), generator=g, device=DEV).mul_(1 / math.sqrt(k)).to(torch.bfloat16)
    b = torch.randn((e, n, r), generator=g, device=DEV).mul_(0.05).to(torch.bfloat16)
    scales = torch.rand(e, generator=g, device=DEV) + 0.5
    x = _act(g, case["tokens"], k, case["x"])
    base = None
    if case["base"] != "none":
        base = torch.randn((case["tokens"], n), generator=g, device=DEV).to(DTYPES[case["base"]])
    return a, b, scales, x, base


# ---------------------------------------------------------------------------
# prepare / run
# ---------------------------------------------------------------------------

def prepare(case, seed):
    return {"sort": _prepare_sort, "adapters": _prepare_adapt}.get(case["kind"], _prepare_move)(
        case, seed)


def run(state):
    return state["run"](state)


def _int(*shape):
    return torch.empty(shape, dtype=torch.int32, device=DEV)


def _prepare_sort(case, seed):
    ids, weights = _sort_inputs(case, seed)
    st = {"run": _run_sort, "case": case, "ids": ids, "weights": weights}
    if own:
        import cascadia_amd as cl
        e, n = case["experts"], ids.numel()
        st["offsets"], st["slots"], st["rows"] = _int(e + 1), _int(n), _int(*ids.shape)
        need = cl.sort_tokens_workspace_bytes(case["tokens"], ids.shape[1], e)
        st["ws"] = torch.empty(max(256, need), dtype=torch.uint8, device=DEV)
    return st


def _run_sort(st):
    c = st["case"]
    if own:
        import cascadia_amd as cl
        k = st["ids"].shape[1]
        w = {"weights": st["weights"], "threshold": THRESHOLD} if c["weights"] else {}
        cl.sort_tokens(st["ids"], k, c["experts"], st["offsets"], st["slots"], st["rows"],
                       workspace=st["ws"], **w)
        return {"offsets": st["offsets"], "slots": st["slots"], "rows": st["rows"]}
    out = _plain_sort(st["ids"], _kept(c, st["ids"], st["weights"]), c["experts"])
    return dict(zip(("offsets", "slots", "rows"), out))


def _prepare_move(case, seed):
    st = _move_inputs(case, seed)
    st["case"], st["k"] = case, st["rows"].shape[1]
    st["run"] = {"gather": _run_gather, "combine": _run_combine, "spread": _run_spread,
                 "grad": _run_grad}[case["kind"]]
    if own:
        t, h, kind = case["tokens"], case["hidden"], case["kind"]
        n = t * st["k"]
        # (rows behind the last one that a slot has stay as they are)
        if kind == "gather":
            st["xs"] = torch.zeros((n, h), dtype=DTYPES[case["y"]], device=DEV)
        elif kind == "grad":
            st["dys"] = torch.zeros_like(st["ys"])
            st["dw"] = torch.empty((t, st["k"]), device=DEV)
        else:
            st["out"] = torch.empty((t, h), dtype=DTYPES[case["y"]], device=DEV)
    return st


def _to_rows(values, rows):
    """values [n, h] to the rows that their slots have; the other rows zero."""
    n = rows.numel()
    at = torch.where(rows < 0, torch.full_like(rows, n), rows).view(-1).long()
    out = torch.zeros((n + 1, values.shape[1]), dtype=values.dtype, device=values.device)
    out[at] = values
    return out[:n]


def _run_gather(st):
    if own:
        import cascadia_amd as cl
        return cl.gather_tokens(st["x"], st["rows"], st["xs"], top_k=st["k"])
    return _to_rows(st["x"].to(DTYPES[st["case"]["y"]]).repeat_interleave(st["k"], 0), st["rows"])


def _slot_values(st):
    """f32 rows of the slots [tokens, k, h], zero for those left out."""
    v = st["ys"][st["rows"].clamp(min=0).long()].float()
    return torch.where((st["rows"] >= 0).unsqueeze(2), v, torch.zeros_like(v))


def _run_combine(st):
    if own:
        import cascadia_amd as cl
        return cl.combine_tokens(st["ys"], st["rows"], st["out"], top_k=st["k"],
                                 weights=st["weights"], residual=st["residual"])
    v = (_slot_values(st) * st["weights"].unsqueeze(2)).sum(1)
    return (st["residual"].float() + v).to(DTYPES[st["case"]["y"]])


def _run_spread(st):
    if own:
        import cascadia_amd as cl
        return cl.gather_tokens_grad(st["ys"], st["rows"], st["out"], top_k=st["k"])
    return _slot_values(st).sum(1).to(DTYPES[st["case"]["y"]])


def _run_grad(st):
    if own:
        import cascadia_amd as cl
        cl.combine_tokens_grad(st["dout"], st["ys"], st["rows"], st["weights"], st["dys"], st["dw"],
                               top_k=st["k"])
        return {"dys": st["dys"], "dweights": st["dw"]}
    dout = st["dout"].float().unsqueeze(1)
    dw = (_slot_values(st) * dout).sum(2)
    dys = (st["weights"].unsqueeze(2) * dout).to(st["ys"].dtype)
    return {"dys": _to_rows(dys.flatten(0, 1), st["rows"]), "dweights": dw}


def _prepare_adapt(case, seed):
    a, b, scales, x, base = _adapt_inputs(case, seed)
    ids, ranks = _requests(case, seed), _ranks(case, seed)
    st = {"run": _run_adapt, "case": case, "x": x, "base": base}
    if own:
        import cascadia_amd as cl
        # (a batch's rows are grouped once for all of its projections)
        ids, t = ids.to(DEV), case["tokens"]
        st["offsets"], st["slots"], rows = _int(case["adapters"] + 1), _int(t), _int(t)
        cl.sort_tokens(ids, 1, case["adapters"], st["offsets"], st["slots"], rows)
        st["adapters"] = cl.Adapters(a, b, scales=scales,
                                     ranks=torch.tensor(ranks, dtype=torch.int32, device=DEV))
        need = cl.adapters_workspace_bytes(st["adapters"], t)
        st["ws"] = torch.empty(max(256, need), dtype=torch.uint8, device=DEV)
        st["ys"] = torch.empty((t, case["n"]), dtype=DTYPES[case["y"]], device=DEV)
        return st
    st["a"], st["b"], st["ranks"] = a, b, ranks
    st["scales"] = scales.tolist()
    st["groups"] = [(i, (ids == i).nonzero().view(-1).to(DEV)) for i in ids.unique().tolist()
                    if i >= 0]
    return st


def _run_adapt(st):
    c = st["case"]
    if own:
        import cascadia_amd as cl
        return cl.adapters_forward(st["adapters"], st["x"], st["offsets"], st["slots"], st["ys"],
                                   base=st["base"], workspace=st["ws"])
    if st["base"] is not None:
        y = st["base"].to(torch.float32, copy=True)
    else:
        y = torch.zeros((c["tokens"], c["n"]), device=DEV)
    for i, at in st["groups"]:
        r = st["ranks"][i]
        inner = st["x"][at].float() @ st["a"][i, :r].float().T
        y[at] += st["scales"][i] * (inner @ st["b"][i, :, :r].float().T)
    return y.to(DTYPES[c["y"]])


# ---------------------------------------------------------------------------
# what one pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    seeds = range(4)
    if case["kind"] == "adapters":
        k, n, t = case["k"], case["n"], case["tokens"]
        b = t * n * (_bytes_of(case["base"]) + _bytes_of(case["y"])) + 4 * t
        flops = 0
        for s in seeds:
            ids, ranks = _requests(case, s), _ranks(case, s)
            for i in ids.unique().tolist():
                if i >= 0:
                    rows = int((ids == i).sum())
                    b += (rows * k * _bytes_of(case["x"]) + 2 * ranks[i] * (k + n)) / 4
                    flops += 2 * rows * ranks[i] * (k + n) / 4
        return {"bytes": b, "flops": flops}
    t, k = case["tokens"], min(case["top_k"], case["experts"])
    if case["kind"] == "sort":
        return {"bytes": t * k * (16 if case["weights"] else 12) + 4 * (case["experts"] + 1),
                "flops": t * k}
    h, kept = case["hidden"], t - case["padded"]
    slots, x, y = kept * k * h, _bytes_of(case["x"]), _bytes_of(case["y"])
    if case["kind"] == "gather":
        return {"bytes": kept * h * x + slots * y + 4 * t * k, "flops": slots}
    if case["kind"] == "combine":
        return {"bytes": slots * x + 2 * t * h * y + 8 * t * k, "flops": 2 * slots}
    if case["kind"] == "spread":
        return {"bytes": slots * x + t * h * y + 4 * t * k, "flops": slots}
    return {"bytes": 2 * slots * x + kept * h * y + 12 * t * k, "flops": 3 * slots}


# ---------------------------------------------------------------------------
# what a pass returns, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    if case["kind"] == "sort":
        return None  # (whole numbers)
    if case["kind"] == "adapters":
        return _exact_adapt(case, seed)
    t = _move_inputs(case, seed)
    rows, w = t["rows"].long(), t["weights"].double()
    tokens, k = rows.shape
    if case["kind"] == "gather":
        out = torch.zeros((tokens * k, case["hidden"]), dtype=torch.float64, device=DEV)
        for j in range(k):
            left = rows[:, j] >= 0
            out.index_copy_(0, rows[left, j], t["x"][left].double())
        return out
    if case["kind"] == "grad":
        dys = torch.zeros(t["ys"].shape, dtype=torch.float64, device=DEV)
        dw = torch.zeros((tokens, k), dtype=torch.float64, device=DEV)
        for j in range(k):
            left = (rows[:, j] >= 0).nonzero().view(-1)
            d, at = t["dout"][left].double(), rows[left, j]
            dys.index_copy_(0, at, d * w[left, j, None])
            dw[left, j] = torch.linalg.vecdot(d, t["ys"][at].double())
        return {"dys": dys, "dweights": dw}
    out = t["residual"].double() if case["kind"] == "combine" else torch.zeros(
        (tokens, case["hidden"]), dtype=torch.float64, device=DEV)
    for j in range(k):
        left = (rows[:, j] >= 0).nonzero().view(-1)
        v = t["ys"][rows[left, j]].double()
        out.index_add_(0, left, v * w[left, j, None] if case["kind"] == "combine" else v)
    return out


def _exact_adapt(case, seed):
    a, b, scales, x, base = _adapt_inputs(case, seed)
    ids, ranks = _requests(case, seed), _ranks(case, seed)
    out = base.double() if base is not None else torch.zeros(
        (case["tokens"], case["n"]), dtype=torch.float64, device=DEV)
    for i in range(case["adapters"]):
        at = torch.nonzero(ids == i, as_tuple=True)[0].to(DEV)
        if at.numel() == 0:
            continue
        inner = torch.matmul(a[i, :ranks[i]].double(), x[at].double().T)
        delta = torch.matmul(b[i, :, :ranks[i]].double(), inner) * scales[i].double()
        out.index_add_(0, at, delta.T)
    return out
