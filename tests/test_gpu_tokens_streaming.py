"""The moves over 256 MiB and more of slots' rows in whole lines (written and read past the
caches), in every pair of types and over several blocks of columns: whole numbers, whose
sums are exact in either type, so that every slot's row counts."""
import pytest
import torch

from test_gpu_adapters import cl, gen  # noqa: F401

pytestmark = pytest.mark.gpu
F32, BF16, U8 = torch.float32, torch.bfloat16, torch.uint8
SIZE = {F32: 4, BF16: 2, U8: 1}
K, E, MOST = 8, 60, 256 << 20


def batch(cl, y_type):
    """tokens, columns (a part of a workgroup's in the last block), rows [T, K]."""
    cols = 8256 if y_type is not U8 else 16512
    T = MOST // (K * cols * SIZE[y_type]) + 3
    assert T * K * cols * SIZE[y_type] >= MOST and cols * SIZE[y_type] % 128 == 0
    g = gen(T)
    ids = torch.rand((T, E), generator=g).topk(K, dim=1).indices.int()
    ids[torch.rand((T, K), generator=g) < 0.05] = -1
    ids[-2:] = -1
    off, slots = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (E + 1, T * K))
    rows = torch.empty((T, K), dtype=torch.int32, device="cuda")
    cl.sort_tokens(ids.cuda(), K, E, off, slots, rows)
    return T, cols, rows


def whole(seed, shape, dtype, most):
    g = torch.Generator(device="cuda").manual_seed(seed)
    low = 0 if dtype is U8 else -most
    return torch.randint(low, most + 1, shape, generator=g, device="cuda", dtype=torch.int16).to(dtype)


def slots_of(rows):
    """(token, choice, row) of the slots that are not left out."""
    t, j = (rows >= 0).nonzero(as_tuple=True)
    return t, j, rows[t, j].long()


@pytest.mark.parametrize("x_type,y_type", [(BF16, BF16), (F32, F32), (F32, BF16), (BF16, F32),
                                           (U8, U8)])
def test_gather(cl, x_type, y_type):
    T, cols, rows = batch(cl, y_type)
    x = whole(1, (T, cols), x_type, 100)
    xs = torch.full((T * K, cols), 111, dtype=y_type, device="cuda")
    cl.gather_tokens(x, rows, xs, top_k=K)
    t, _, r = slots_of(rows)
    left = torch.ones(T * K, dtype=torch.bool, device="cuda")
    left[r] = False
    assert torch.equal(xs[r], x[t].to(y_type))
    assert int(left.sum()) > 0 and bool((xs[left] == 111).all())


@pytest.mark.parametrize("y_type,out_type", [(BF16, BF16), (F32, F32), (F32, BF16), (BF16, F32)])
def test_combine(cl, y_type, out_type):
    T, cols, rows = batch(cl, y_type)
    ys = whole(2, (T * K, cols), y_type, 7)
    w = whole(3, (T, K), F32, 3)
    w[w == 0] = 2.0
    res = whole(4, (T, cols), out_type, 20)
    out = torch.empty_like(res)
    cl.combine_tokens(ys, rows, out, top_k=K, weights=w, residual=res)
    dx = torch.empty_like(res)
    cl.gather_tokens_grad(ys, rows, dx, top_k=K)
    want, plain = res.float(), torch.zeros((T, cols), device="cuda")
    for j in range(K):
        at = (rows[:, j] >= 0).nonzero().view(-1)
        v = ys[rows[at, j].long()].float()
        want[at] += w[at, j, None] * v
        plain[at] += v
    assert float(want.abs().max()) <= 256  # (whole in bf16 as well)
    assert torch.equal(out.float(), want) and torch.equal(dx.float(), plain)


@pytest.mark.parametrize("y_type,d_type", [(BF16, BF16), (F32, F32), (F32, BF16), (BF16, F32)])
@pytest.mark.parametrize("inplace", [False, True])
def test_combine_grad(cl, y_type, d_type, inplace):
    T, cols, rows = batch(cl, y_type)
    ys = whole(5, (T * K, cols), y_type, 7)
    w = whole(6, (T, K), F32, 3)
    dout = whole(7, (T, cols), d_type, 20)
    t, j, r = slots_of(rows)
    want_dw = torch.zeros((T, K), device="cuda")
    for i in range(K):
        at = (rows[:, i] >= 0).nonzero().view(-1)
        want_dw[at, i] = (ys[rows[at, i].long()].float() * dout[at].float()).sum(1)
    left = torch.ones(T * K, dtype=torch.bool, device="cuda")
    left[r] = False
    dys = ys if inplace else torch.full_like(ys, 111)
    behind = dys[left].clone()
    dw = torch.empty_like(w)
    cl.combine_tokens_grad(dout, ys, rows, w, dys, dw, top_k=K)
    assert torch.equal(dw, want_dw)
    assert torch.equal(dys[r].float(), w[t, j, None] * dout[t].float())
    assert torch.equal(dys[left], behind)
