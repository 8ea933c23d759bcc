"""Adapter cases whose outputs have tight bounds however long the rows are, and the
checks on them (CPU; the kernels' inputs and outputs are passed in and out).

  whole   small whole numbers: every sum is exact in f32 in any order, so are outputs
  picks   each rank picks one column of full f32 values, another in every block of 128
          columns: three bf16 planes hold a value whole, and each of the two sums of
          three may truncate by 2^-23 of it
  normal  random values, by the relative L2 error of all adapters' outputs: an addition
          is off by 2^-23 of a partial sum at most (a matrix core may truncate), and
          independent errors of 3 n additions to partial sums that grow as their square
          root come to 2^-23 sqrt(3 n / 2) of the sum
"""
import numpy as np
import torch

F32, BF16 = torch.float32, torch.bfloat16
BLOCK = 128  # columns

# T, E, R, K, N: K in several slices, tails in K, one to four tiles of 16 rows
SHAPES = [
    (1, 1, 16, 4096, 80), (3, 4, 16, 14336, 130), (16, 2, 8, 1032, 64), (64, 20, 64, 4096, 200),
    (40, 3, 128, 7168, 96), (257, 6, 32, 7168, 96), (300, 300, 16, 2056, 72), (500, 9, 48, 1288, 64),
    (1030, 3, 16, 4096, 68), (1100, 4, 32, 4104, 64), (1100, 3, 64, 4168, 64), (2100, 3, 64, 4104, 64),
    (2100, 5, 128, 4096, 64), (2500, 900, 24, 2056, 64), (4096, 9, 32, 4096, 64)]


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def rows(g, T, E):
    ids = torch.randint(-1, E, (T,), generator=g, dtype=torch.int32)
    ids[0] = E - 1
    return ids


def whole(T, E, R, K, N, x_type):
    """a, b, ids, x, base (f32): whole numbers of at most 2, ranks' sums below 2^24."""
    assert 4 * K * 2 * R < 2 ** 24
    g = gen(T + K + R)

    def some(*shape):
        return torch.randint(-2, 3, shape, generator=g, dtype=torch.int8).float()

    return (some(E, R, K).to(BF16), some(E, N, R).to(BF16), rows(g, T, E), some(T, K).to(x_type),
            some(T, N))


def picked(R, K, E):
    """The column of each adapter's rank: a column of another block each, in turn over all
    blocks, the last one's last column among them."""
    blocks = -(-K // BLOCK)
    at = torch.arange(E * R)
    cols = at % blocks * BLOCK + at * 37 % BLOCK
    cols = torch.where(cols < K, cols, K - 1 - at % 8)
    cols[blocks - 1 if blocks <= E * R else -1] = K - 1
    return cols.view(E, R)


def picks(T, E, R, K, N):
    """a, b, ids, x, base (0): outputs are columns of x."""
    g = gen(T + K + R + 1)
    cols = picked(R, K, E)
    a, b = torch.zeros((E, R, K), dtype=BF16), torch.zeros((E, N, R), dtype=BF16)
    a[torch.arange(E)[:, None], torch.arange(R), cols] = 1.0
    b[:, torch.arange(N), torch.arange(N) % R] = 1.0
    x = torch.randn((T, K), generator=g)
    return a, b, rows(g, T, E), x, torch.zeros((T, N))


def normal(T, E, R, K, N, x_type):
    g = gen(T + K + R + 2)
    a = (torch.randn((E, R, K), generator=g) / K ** 0.5).to(BF16)
    b = (torch.randn((E, N, R), generator=g) / R ** 0.5).to(BF16)
    return a, b, rows(g, T, E), torch.randn((T, K), generator=g).to(x_type), torch.zeros((T, N))


def exact(case, x=None):
    """The outputs in 64 bits, [T, N] (x: other rows in place of the case's)."""
    a, b, ids, own, base = case
    x = own if x is None else x
    out = base.double()
    for i in range(a.shape[0]):
        at = (ids == i).nonzero().view(-1)
        if at.numel():
            out[at] += x[at].double() @ a[i].double().T @ b[i].double().T
    return out


def whole_ok(got, case):
    return torch.equal(got, exact(case).to(got.dtype))


def picks_ok(got, case):
    want = exact(case)
    bound = (2.0 ** -21 + (2.0 ** -8 if got.dtype is BF16 else 0)) * want.abs()
    return bool(((got.double() - want).abs() <= bound).all())


def normal_ok(got, case):
    want = exact(case)
    K, R = case[3].shape[1], case[0].shape[1]
    bound = 2.0 ** -23 * ((1.5 * K) ** 0.5 + (1.5 * R) ** 0.5 + 4)
    if got.dtype is BF16:
        bound += 2.0 ** -8
    return float((got.double() - want).norm() / want.norm()) <= bound


def planes(x, n):
    """x as the sum of its first n bf16 planes (the first truncated)."""
    out, rest = torch.zeros_like(x), x.clone()
    for i in range(n):
        p = (rest.view(torch.int32) & -65536).view(F32) if i == 0 else rest.to(BF16).float()
        out, rest = out + p, rest - p
    return out
