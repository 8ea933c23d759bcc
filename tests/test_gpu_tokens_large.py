"""Many rows, wide buffers, two streams at once and graphs over the library's own
workspace: sorting, moves and adapters against 64-bit products on the GPU."""
import threading

import pytest
import torch

import tokens_ref as ref
from test_gpu_adapters import cl, gen, plan  # noqa: F401
from test_gpu_tokens import some_ids

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def case(T, E, R, K, N, x_type, base_type, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    a, b = (normal(E, R, K) / K ** 0.5).to(BF16), (normal(E, N, R) / R ** 0.5).to(BF16)
    ids = torch.randint(-1, E, (T,), generator=g, device="cuda", dtype=torch.int32)
    return a, b, ids, normal(T, K).to(x_type), normal(T, N).to(base_type)


def check(a, b, ids, x, base, ys):
    """ys against 64 bits, adapter by adapter, within the bound of tokens_ref.adapters
    (scales 1, all ranks)."""
    E, R, K = a.shape
    bf16 = ys.dtype is BF16
    plane = 2.0 ** -16 if bf16 else 2.0 ** -24
    for i in range(-1, E):
        at = (ids == i).nonzero().view(-1)
        out = base[at].double()
        bound = torch.zeros_like(out)
        if i >= 0:
            A, B, xt = a[i].double(), b[i].double(), x[at].double()
            u = xt @ A.T
            du = ((3 * K + 64) * 2 * ref.U32 + 2 * ref.U32) * (xt.abs() @ A.abs().T)
            du = du + (2 * ref.U32 + plane) * (u.abs() + du)
            out = out + u @ B.T
            bound = du @ B.abs().T + (3 * R + 8) * 2 * ref.U32 * (u.abs() @ B.abs().T)
        bound = bound + 2 * ref.U32 * (out.abs() + bound)
        bound = bound + (ref.BF16 if bf16 else ref.U32) * (out.abs() + bound) + 1e-37
        assert bool(((ys[at].double() - out).abs() <= bound).all()), i


@pytest.mark.parametrize("T,E,R,K,N,x_type,y_type", [
    (4200, 5, 32, 264, 8256, BF16, BF16), (4200, 5, 16, 264, 8250, F32, BF16),
    (2100, 3, 64, 520, 8256, F32, F32), (2100, 3, 128, 520, 8256, BF16, F32),
    (70001, 3, 16, 72, 40, F32, F32), (70001, 1000, 8, 72, 40, BF16, BF16)])
def test_adapters_over_many_rows(cl, T, E, R, K, N, x_type, y_type):
    """Outputs past the caches (64 MiB and more, in whole lines and not), many chunks."""
    a, b, ids, x, base = case(T, E, R, K, N, x_type, y_type)
    off, slots = plan(cl, ids, E)
    A = cl.Adapters(a, b)
    ys = torch.empty_like(base)
    cl.adapters_forward(A, x, off, slots, ys, base=base)
    check(a, b, ids, x, base, ys)
    # in place: the same bits
    both = base.clone()
    cl.adapters_forward(A, x, off, slots, both, base=both)
    assert torch.equal(both, ys)


def test_adapters_in_buffers_past_4_gib(cl):
    """Rows that lie so far apart that the last ones are past 2^32 bytes."""
    T, E, R, K, N, wide = 20000, 3, 16, 64, 96, 110000
    a, b, ids, x, base = case(T, E, R, K, N, BF16, BF16)
    buf = torch.empty((T, wide), dtype=BF16, device="cuda")
    assert T * wide * 2 > 2 ** 32
    xs, ys = buf[:, :K], buf[:, wide - N:]
    xs.copy_(x)
    ys.copy_(base)
    buf[:, K:wide - N].zero_()
    off, slots = plan(cl, ids, E)
    cl.adapters_forward(cl.Adapters(a, b), xs, off, slots, ys, base=ys)
    check(a, b, ids, x, base, ys)
    assert torch.equal(xs, x) and not buf[:, K:wide - N].any()


def test_two_streams_over_the_librarys_workspace(cl):
    """Calls without a workspace from two threads, each on a stream of its own."""
    jobs = []
    for s in range(2):
        T, E, R, K, N = 300 + 77 * s, 20, 32, 1032, 520
        a, b, ids, x, base = case(T, E, R, K, N, F32, F32, seed=s)
        big = some_ids(gen(s), 9000, 8, 300).cuda()
        jobs.append((a, b, ids, x, base, big))

    def call(j):
        a, b, ids, x, base, big = j
        E, n = a.shape[0], big.numel()
        off, slots = plan(cl, ids, E)
        y = cl.adapters_forward(cl.Adapters(a, b), x, off, slots, torch.empty_like(base), base=base)
        out = [torch.empty(m, dtype=torch.int32, device="cuda") for m in (301, n, n)]
        cl.sort_tokens(big, 8, 300, *out)
        return [y] + out

    want = [call(j) for j in jobs]
    torch.cuda.synchronize()
    bad = []

    def run(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(20):
                got = call(jobs[i])
                st.synchronize()
                if not all(torch.equal(p, q) for p, q in zip(got, want[i])):
                    bad.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_recorded_without_a_workspace(cl):
    """The library's buffer for graphs, grown by the eager call before; two graphs that use
    it run one after the other."""
    a, b, ids, x, base = case(500, 9, 32, 1032, 264, BF16, BF16)
    big = some_ids(gen(5), 9000, 8, 300).cuda()
    n = big.numel()
    off, slots, rows = (torch.empty(m, dtype=torch.int32, device="cuda") for m in (301, n, n))
    aoff, aslots = plan(cl, ids, 9)
    A, y = cl.Adapters(a, b), torch.empty_like(base)

    def sort():
        cl.sort_tokens(big, 8, 300, off, slots, rows)

    def adapt():
        cl.adapters_forward(A, x, aoff, aslots, y, base=base)

    sort(), adapt()
    want = [t.clone() for t in (off, slots, rows, y)]
    torch.cuda.synchronize()
    graphs = []
    for f in (sort, adapt):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            f()
    for _ in range(3):
        for t in (off, slots, rows, y):
            t.zero_()
        for graph in graphs:
            graph.replay()
            sort(), adapt()  # eager calls beside: their own buffer
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip((off, slots, rows, y), want))


def test_the_largest_batch(cl):
    """2^20 tokens (the limit): sorted, moved and added back."""
    T, k, E, cols = 1 << 20, 3, 1024, 4
    g = torch.Generator(device="cuda").manual_seed(8)
    ids = torch.randint(0, E + 20, (T, k), generator=g, device="cuda", dtype=torch.int32)
    off, slots, rows = (torch.empty(m, dtype=torch.int32, device="cuda") for m in (E + 1, T * k, T * k))
    cl.sort_tokens(ids, k, E, off, slots, rows)
    key = torch.where(ids < E, ids, E).view(-1)
    assert torch.equal(slots.long(), torch.sort(key, stable=True).indices)
    n = int(off[-1])
    assert n == int((ids < E).sum()) and torch.equal(rows[slots[:n].long()], torch.arange(n, device="cuda").int())
    assert bool((rows[slots[n:].long()] == -1).all())
    x = torch.randint(-8, 9, (T, cols), generator=g, device="cuda").float()
    xs = torch.zeros((T * k, cols), device="cuda")
    rows = rows.view(T, k)
    cl.gather_tokens(x, rows, xs, top_k=k)
    out = torch.empty_like(x)
    cl.gather_tokens_grad(xs, rows, out, top_k=k)
    assert torch.equal(out, x * (ids < E).sum(1, keepdim=True))
    dw = torch.empty((T, k), device="cuda")
    cl.combine_tokens_grad(x, xs, rows, torch.ones((T, k), device="cuda"), xs, dw, top_k=k)
    assert torch.equal(dw, (ids < E) * (x * x).sum(1, keepdim=True))
