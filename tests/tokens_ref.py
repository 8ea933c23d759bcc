"""64-bit reference of the sorting of tokens by expert, of the moves there and back and
of low-rank adapters (numpy, on the CPU), with bounds on what 32-bit arithmetic may
add."""
import numpy as np

U32 = 2.0 ** -24   # half a step of f32, relative
BF16 = 2.0 ** -8   # half a step of bf16, relative


def sort(ids, n_experts, weights=None, threshold=0.0):
    """(offsets, slots, rows) from the definition, slot by slot."""
    flat = np.asarray(ids).reshape(-1)
    w = None if weights is None else np.asarray(weights, np.float32).reshape(-1)
    groups = [[] for _ in range(n_experts + 1)]
    for i, e in enumerate(flat.tolist()):
        out = not 0 <= e < n_experts or (w is not None and bool(w[i] < np.float32(threshold)))
        groups[n_experts if out else e].append(i)
    offsets = np.cumsum([0] + [len(g) for g in groups[:n_experts]]).astype(np.int32)
    slots = np.array([i for g in groups for i in g], np.int32)
    rows = np.full(flat.size, -1, np.int32)
    kept = slots[:offsets[-1]]
    rows[kept] = np.arange(kept.size)
    return offsets, slots, rows.reshape(np.asarray(ids).shape)


def gather(x, rows, xs):
    """xs with the slots' rows of x (a copy)."""
    out = np.array(xs)
    for t, j in np.argwhere(rows >= 0):
        out[rows[t, j]] = x[t]
    return out


def combine(ys, rows, weights, residual, out_bf16):
    """(out, bound): the bound counts a rounding of each partial sum (f32, one per
    slot and one with the residual) and the output's."""
    T, k = rows.shape
    out = np.zeros((T, ys.shape[1])) if residual is None else np.array(residual, np.float64)
    total = np.abs(out)
    for t, j in np.argwhere(rows >= 0):
        v = ys[rows[t, j]].astype(np.float64) * (1.0 if weights is None else float(weights[t, j]))
        out[t] += v
        total[t] += np.abs(v)
    bound = (k + 1) * U32 * (1 + 1e-5) * total
    return out, bound + (BF16 if out_bf16 else U32) * (np.abs(out) + bound)


def combine_grad(dout, ys, rows, weights, dys, y_bf16):
    """(dys, its bound, dweights, its bound): a product rounds once to f32 and once to
    dys's type; a dot product's cols terms are added in some order."""
    out, bound = np.array(dys, np.float64), np.zeros(dys.shape)
    dw, dwb = np.zeros(rows.shape), np.zeros(rows.shape)
    for t, j in np.argwhere(rows >= 0):
        r, d = rows[t, j], dout[t].astype(np.float64)
        v = d * float(weights[t, j])
        out[r] = v
        bound[r] = (U32 + (BF16 if y_bf16 else 0)) * (1 + 1e-5) * np.abs(v)
        p = ys[r].astype(np.float64) * d
        dw[t, j] = p.sum()
        dwb[t, j] = (p.size + 1) * U32 * (1 + 1e-3) * np.abs(p).sum()
    return out, bound + 1e-45, dw, dwb + 1e-45


def adapters(a, b, ranks, scales, ids, x, base, y_bf16):
    """(ys, bound).  Products of bf16 values are exact in f32; a sum of n of them, in
    some order, is off by 2^-23 of the terms' magnitudes each (a matrix core may
    truncate).  f32 x enters as three bf16 values that hold it, the inner values as three
    that hold them to 2^-24 (f32 y) or two (2^-16)."""
    T, N, K = len(ids), b.shape[1], a.shape[2]
    out = np.zeros((T, N)) if base is None else np.array(base, np.float64)
    bound = np.zeros((T, N))
    plane = 2.0 ** -16 if y_bf16 else 2.0 ** -24
    for t, i in enumerate(np.asarray(ids).tolist()):
        if not 0 <= i < a.shape[0]:
            continue
        r, s = int(ranks[i]), float(scales[i])
        A, B = a[i, :r].astype(np.float64), b[i, :, :r].astype(np.float64)
        xt = x[t].astype(np.float64)
        u = A @ xt
        du = ((3 * K + 64) * 2 * U32 + 2 * U32) * (np.abs(A) @ np.abs(xt))
        su = s * u
        dsu = abs(s) * du + (2 * U32 + plane) * (np.abs(su) + abs(s) * du)
        out[t] += B @ su
        bound[t] = np.abs(B) @ dsu + (3 * r + 8) * 2 * U32 * (np.abs(B) @ np.abs(su))
    bound += 2 * U32 * (np.abs(out) + bound)
    return out, bound + (BF16 if y_bf16 else U32) * (np.abs(out) + bound) + 1e-37
