"""adapters_forward at the sizes that the header allows: whole numbers and picked columns,
whose outputs are exact."""
import pytest
import torch

from test_gpu_adapters import cl  # noqa: F401

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def whole(seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-2, 3, shape, generator=g, device="cuda", dtype=torch.int8).to(BF16)


def plan(cl, ids, E):
    T = ids.numel()
    off, slots, rows = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (E + 1, T, T))
    cl.sort_tokens(ids, 1, E, off, slots, rows)
    return off, slots


def exact(a, b, ids, x, base):
    """(f32 matrix products of whole numbers below 2^24: exact)"""
    out = base.float().clone()
    for i in range(a.shape[0]):
        at = (ids == i).nonzero().view(-1)
        out[at] += x[at].float() @ a[i].float().T.contiguous() @ b[i].float().T.contiguous()
    return out


@pytest.mark.parametrize("E", [1, 7])
def test_rows_2_to_the_20(cl, E):
    T, R, K, N = 1 << 20, 8, 16, 24
    a, b, x, base = whole(1, E, R, K), whole(2, E, N, R), whole(3, T, K), whole(4, T, N)
    ids = torch.randint(-1, E, (T,), device="cuda", dtype=torch.int32)
    y = torch.empty((T, N), device="cuda")
    cl.adapters_forward(cl.Adapters(a, b), x, *plan(cl, ids, E), y, base=base)
    assert torch.equal(y, exact(a, b, ids, x, base))
    with pytest.raises(cl.CascadiaInt4Error):
        more = torch.zeros(T + 1, dtype=torch.int32, device="cuda")
        cl.adapters_forward(cl.Adapters(a, b), torch.zeros((T + 1, K), dtype=BF16, device="cuda"),
                            torch.zeros(E + 1, dtype=torch.int32, device="cuda"), more,
                            torch.empty((T + 1, N), device="cuda"))


@pytest.mark.parametrize("x_type", [BF16, F32])
def test_columns_2_to_the_20_and_rank_256(cl, x_type):
    T, R, K, N = 19, 256, 1 << 20, 300
    a, x = whole(5, 1, R, K), whole(6, T, K)
    b = torch.zeros((1, N, R), dtype=BF16, device="cuda")
    b[0, torch.arange(N), torch.arange(N) % R] = 1.0
    ids = torch.zeros(T, dtype=torch.int32, device="cuda")
    y = torch.empty((T, N), device="cuda")
    cl.adapters_forward(cl.Adapters(a, b), x.to(x_type), *plan(cl, ids, 1), y)
    u = x.float() @ a[0].float().T.contiguous()
    assert float(u.abs().max()) < 2 ** 24
    assert torch.equal(y, u[:, torch.arange(N) % R])


@pytest.mark.parametrize("y_type", [BF16, F32])
def test_outputs_2_to_the_22(cl, y_type):
    T, R, K, N = 5, 8, 64, 1 << 22
    a, b, x, base = whole(7, 2, R, K), whole(8, 2, N, R), whole(9, T, K), whole(10, T, N)
    ids = torch.tensor([1, -1, 0, 1, 0], dtype=torch.int32, device="cuda")
    y = torch.empty((T, N), dtype=y_type, device="cuda")
    cl.adapters_forward(cl.Adapters(a, b), x, *plan(cl, ids, 2), y, base=base)
    assert torch.equal(y, exact(a, b, ids, x, base).to(y_type))


def test_strides_of_2_to_the_29(cl):
    T, R, K, N, ld = 3, 8, 72, 100, 1 << 29
    a, b, x, base = whole(11, 2, R, K), whole(12, 2, N, R), whole(13, T, K), whole(14, T, N).float()
    ids = torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda")
    buf = torch.empty(2 * ld + 1024, device="cuda")
    xs, ys = buf.as_strided((T, K), (ld, 1)), buf.as_strided((T, N), (ld, 1), 512)
    xs.copy_(x)
    ys.copy_(base)
    A = cl.Adapters(a, b)
    cl.adapters_forward(A, xs, *plan(cl, ids, 2), ys, base=ys)
    assert torch.equal(ys, exact(a, b, ids, x, base))
    wide = buf.as_strided((2, K), (ld + 8, 1))
    with pytest.raises(cl.CascadiaInt4Error):
        cl.adapters_forward(A, wide, *plan(cl, ids[:2].contiguous(), 2), ys[:2], base=ys[:2])
