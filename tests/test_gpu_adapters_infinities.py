"""adapters_forward where a or b has infinities: what the formula gives, although f32 values
enter the products in planes."""
import numpy as np
import pytest
import torch

from test_gpu_adapters import case, cl, gen, host, plan  # noqa: F401
from test_gpu_adapters_bits import bits, forward

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
INF, NAN = float("inf"), float("nan")


def products(w, v):
    """w @ v in 64 bits: infinite where infinite terms agree in sign, NaN where they do not
    or where one is 0 * inf."""
    with np.errstate(invalid="ignore"):
        return (w * v).sum(-1)


@pytest.mark.parametrize("x_type,y_type", [(BF16, BF16), (F32, F32), (F32, BF16), (BF16, F32)])
@pytest.mark.parametrize("T,K", [(12, 264), (60, 264), (60, 4104), (1100, 264), (2100, 264)])
@pytest.mark.parametrize("R", [16, 40, 72])
def test_infinities_of_the_weights(cl, x_type, y_type, T, K, R):
    """Infinities and NaN of a and b against infinite, zero, ordinary and subnormal values:
    what the formula gives.  (Small whole numbers elsewhere, whose sums are exact.)"""
    N, E = 70, 6
    g = gen(23)

    def whole(*shape):
        return torch.randint(-2, 3, shape, generator=g).float()

    a, b, x = whole(E, R, K), whole(E, N, R), whole(T, K)
    x[:, 5] = torch.tensor([1.0, -2.0, 3.0, 0.5])[torch.arange(T) // E % 4]
    for i, r in ((0, 0), (1, R // 2), (2, R - 1)):  # an infinite inner value each
        a[i, r, 5] = -INF if i == 1 else INF
        b[i, :, r] = 1.0 - 2.0 * (torch.arange(N) % 2)
    a[1, R // 2, K - 1] = INF   # where x agrees in sign: NaN
    x[:, K - 1] = 1.0
    b[3, 0, 3], b[3, 1, R - 1], b[3, 2, 0], b[3, 69, 8] = INF, -INF, NAN, INF
    b[3, 3, 3], b[3, 3, R - 1] = INF, -INF
    a[4, 0, 5], b[4, :, 0], b[4, 1, 0], b[4, 2, 0] = INF, 2.0, -INF, 0.0
    a[5, 1, 9], b[5, :, 1] = NAN, 1.0
    x[0, 5], x[1, 5], x[2, 5], x[3, 5] = 0.0, -2.0 ** -10, INF, INF
    x[6, 5], x[7, 5], x[8, 5], x[9, 8] = 2.0 ** -133, -INF, -2.0 ** -126, NAN
    x = x.to(x_type)
    ids = torch.arange(T, dtype=torch.int32) % E
    c = (a.to(BF16), b.to(BF16), torch.full((E,), R, dtype=torch.int32), torch.ones(E), ids, x, None)
    got = host(forward(cl, c, y_type))
    A, B, X = host(c[0]), host(c[1]), host(x)
    for i in range(E):
        at = np.flatnonzero(ids.numpy() == i)
        u = np.stack([products(A[i], X[t]) for t in at])
        want = np.stack([products(B[i], v) for v in u])
        special = ~np.isfinite(want)
        assert np.array_equal(got[at][special], want[special], equal_nan=True), i
        with np.errstate(invalid="ignore"):
            bound = 2.0 ** -20 * np.stack([(np.abs(B[i]) * np.abs(v)).sum(-1) for v in u])
            if y_type is BF16:
                bound = bound + 2.0 ** -8 * np.abs(want)
            assert np.all((np.abs(got[at] - want) <= bound)[~special]), i


@pytest.mark.parametrize("x_type,y_type", [(F32, F32), (F32, BF16), (BF16, F32)])
@pytest.mark.parametrize("T", [2, 33, 1100, 2100])
def test_one_infinite_weight_alone(cl, x_type, y_type, T):
    """An infinity of a reaches its rank's outputs, one of b its own, with its sign."""
    K, N, R = 136, 70, 40
    a, b = torch.zeros((2, R, K)), torch.zeros((2, N, R))
    a[0, 3, 9], b[0, :, 3] = INF, -1.0        # u = inf at rank 3
    a[1, 3, 9], b[1, 5, 3], b[1, 6, 3] = 0.5, INF, 2.0
    x = torch.ones((T, K))
    x[1] = -1.0
    ids = torch.arange(T, dtype=torch.int32) % 2
    for i in (0, 1):  # ranks 0 to 3 only, of which three are zero in a, b and so in u
        c = (a[i:i + 1, 3:11].contiguous().to(BF16), b[i:i + 1, :, 3:11].contiguous().to(BF16),
             torch.ones(1, dtype=torch.int32), torch.ones(1), torch.where(ids == i, 0, -1).int(),
             x.to(x_type), None)
        got = forward(cl, c, y_type).cpu().float()
        at = ids == i
        sign = x[:, 0][at]
        want = torch.full((int(at.sum()), N), -INF) * sign[:, None]
        if i == 1:
            want = torch.zeros_like(want)
            want[:, 5], want[:, 6] = sign * INF, sign
        assert torch.equal(got[at], want)
        assert not got[~at].any()


@pytest.mark.parametrize("T", [1, 20, 1100, 2100])
@pytest.mark.parametrize("nan", [0x7F800001, 0x7FC00000, -0x7FFF01, 0x7FFFFFFF])
def test_every_nan_of_x_stays_one(cl, T, nan):
    """Signalling ones too, whose upper half alone would be an infinity."""
    K, N, R = 136, 70, 40
    g = gen(24)
    a, b = (torch.rand(s, generator=g).to(BF16) + 1.0 for s in ((1, R, K), (1, N, R)))
    x = torch.randn((T, K), generator=g)
    x.view(torch.int32)[T // 2, 9] = nan
    c = (a, b, torch.tensor([R], dtype=torch.int32), torch.ones(1), torch.zeros(T, dtype=torch.int32), x,
         None)
    got = forward(cl, c, F32).cpu()
    assert bool(got[T // 2].isnan().all())
    got[T // 2] = 0
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("R", [16, 40, 72])
def test_in_place_where_sums_are_taken_again(cl, t, R):
    """Rows with infinite sums in either tile of a chunk, over base: as out of place, and
    the rows between them as without any infinity."""
    T, E, K, N = 150, 2, 136, 330
    a, b, ranks, scales, ids, x, base = case(25, T, E, R, K, N, t, t, mixed=False, bare=0.1)
    clean = forward(cl, (a, b, ranks, scales, ids, x, base), t)
    hit = torch.zeros(T, dtype=torch.bool)
    hit[::9] = True
    hit &= (ids >= 0) & (ids < E)
    x = x.clone()
    x[hit, 3], x[hit, 4] = INF, -INF
    out = forward(cl, (a, b, ranks, scales, ids, x, base), t)
    off, slots = plan(cl, ids, E)
    A = cl.Adapters(a.cuda(), b.cuda(), ranks=ranks.cuda(), scales=scales.cuda())
    y = base.cuda()
    cl.adapters_forward(A, x.cuda(), off, slots, y, base=y)
    assert torch.equal(bits(y), bits(out))
    assert torch.equal(bits(out)[~hit], bits(clean)[~hit])
    assert not out.cpu()[hit].isfinite().any()
