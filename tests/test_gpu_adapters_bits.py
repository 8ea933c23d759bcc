"""What adapters_forward keeps of its values: the bits of the inner values, rows without
an adapter as they are."""
import numpy as np
import pytest
import torch

from test_gpu_adapters import case, cl, gen, host, plan  # noqa: F401

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def forward(cl, c, y_type, base=None):
    a, b, ranks, scales, ids, x, own_base = c
    off, slots = plan(cl, ids, a.shape[0])
    A = cl.Adapters(a.cuda(), b.cuda(), ranks=ranks.cuda(), scales=scales.cuda())
    base = own_base if base is None else base
    ys = torch.full((len(ids), b.shape[1]), 77.0, dtype=y_type, device="cuda")
    return cl.adapters_forward(A, x.cuda(), off, slots, ys, base=None if base is None else base.cuda())


@pytest.mark.parametrize("T,E,R,K,N", [(1, 3, 16, 128, 64), (17, 9, 40, 520, 65), (65, 2, 64, 512, 129),
                                       (300, 7, 128, 392, 47), (64, 100, 64, 4096, 2050),
                                       (1030, 3, 32, 2056, 320)])
@pytest.mark.parametrize("x_type", [BF16, F32])
@pytest.mark.parametrize("base_type", [None, BF16, F32])
def test_bf16_outputs_are_the_f32_ones_rounded_once(cl, T, E, R, K, N, x_type, base_type):
    """The same sums whatever ys's type: the outputs differ by its rounding alone."""
    c = case(T + R, T, E, R, K, N, x_type, base_type)
    assert torch.equal(forward(cl, c, BF16), forward(cl, c, F32).to(BF16))


@pytest.mark.parametrize("T", [5, 300])
def test_a_base_that_cancels_the_adapter(cl, T):
    """Adapters that pick columns of f32 x, and a base that takes away its upper 16 bits:
    what is left over comes out to bf16.  (Three planes hold a value whole; each of the
    two sums of three may truncate by 2^-23 of it.)"""
    K, N, R = 264, 96, 24
    g = gen(21)
    cols = torch.randperm(K, generator=g)[:R]
    a, b = torch.zeros((1, R, K), dtype=BF16), torch.zeros((1, N, R), dtype=BF16)
    a[0, torch.arange(R), cols] = 1.0
    b[0, torch.arange(N), torch.arange(N) % R] = 1.0
    x = torch.randn((T, K), generator=g)
    picked = x[:, cols][:, torch.arange(N) % R].contiguous()
    base = -(picked.view(torch.int32) & ~0xFF).view(F32)
    c = (a, b, torch.tensor([R], dtype=torch.int32), torch.ones(1), torch.zeros(T, dtype=torch.int32), x,
         base)
    want = host(base) + host(picked)
    bound = 2.0 ** -8 * np.abs(want) + 2.0 ** -21 * np.abs(host(picked))
    assert np.all(np.abs(host(forward(cl, c, BF16)) - want) <= bound)


def bits(t):
    return t.view(torch.int16 if t.dtype is BF16 else torch.int32).cpu()


@pytest.mark.parametrize("base_type", [F32, BF16])
@pytest.mark.parametrize("y_type", [F32, BF16])
@pytest.mark.parametrize("rank_zero", [False, True])
def test_rows_without_an_adapter_keep_every_bit(cl, base_type, y_type, rank_zero):
    """Zeros of either sign, subnormal values, infinities and the largest values, beside rows
    that have an adapter; out of place and in place."""
    T, E, N, K, R = 75, 3, 104, 64, 16
    g = gen(22)
    a, b = torch.randn((E, R, K), generator=g).to(BF16), torch.randn((E, N, R), generator=g).to(BF16)
    ranks = torch.tensor([R, 0, 8], dtype=torch.int32)
    ids = torch.arange(T, dtype=torch.int32) % E
    if not rank_zero:
        ids[ids == 1] = -1
    bare = (ids == 1) | (ids < 0)
    v = torch.tensor([-0.0, 0.0, -1e-40, 1.0, float("-inf"), 3.3e38, -1.1754944e-38, 0.1])
    base = v[torch.randint(0, 8, (T, N), generator=g)].to(base_type)
    base[~bare] = 0.5
    x = torch.randn((T, K), generator=g).to(BF16)
    c = (a, b, ranks, torch.ones(E), ids, x, base)
    out = forward(cl, c, y_type)
    assert torch.equal(bits(out)[bare], bits(base.to(y_type))[bare])
    assert bool((out.cpu()[~bare] != 0.5).any(1).all())
    if base_type is y_type:
        off, slots = plan(cl, ids, E)
        A = cl.Adapters(a.cuda(), b.cuda(), ranks=ranks.cuda())
        y = base.cuda()
        cl.adapters_forward(A, x.cuda(), off, slots, y, base=y)
        assert torch.equal(bits(y), bits(out))


def test_rows_without_an_adapter_over_many_rows(cl):
    """The same where whole lines are written past the caches."""
    T, E, N, K, R = 9000, 3, 4096, 16, 8
    ids = torch.arange(T, dtype=torch.int32) % 4 - 1
    bare = ids < 0
    x, a, b = torch.ones((T, K)), torch.ones((E, R, K), dtype=BF16), torch.ones((E, N, R), dtype=BF16)
    base = torch.full((T, N), -0.0)
    c = (a, b, torch.full((E,), R, dtype=torch.int32), torch.ones(E), ids, x, base)
    for t in (F32, BF16):
        out = forward(cl, c, t).cpu()
        assert bool((bits(out)[bare] == bits(base[:1].to(t))).all())
        assert bool((out[~bare] == K * R).all())
