"""A product that needs no workspace asks the library for none: recorded into a graph
in a fresh process, where the library holds no memory for graphs yet, its replays give
the eager result."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

SCRIPT = r"""
import sys
sys.path.insert(0, sys.argv[1])
import torch
import cascadia_amd as cl
g = torch.Generator().manual_seed(1)
def codes(*s): return (torch.randn(s, generator=g) * 100).clamp_(-448, 448).to(torch.float8_e4m3fn).cuda()
def case(m, n, k):
    w, x = codes(n, k), codes(m, k)
    ws = torch.rand((-(-n // 128), -(-k // 128)), generator=g).cuda()
    return w, ws, x, torch.rand((m, -(-k // 128)), generator=g).cuda()
def record(m, n, k, dtype, workspace=None):
    w, ws, x, xs = case(m, n, k)
    y = torch.empty((m, n), dtype=dtype, device="cuda")
    call = lambda: cl.fp8_gemm(w, ws, x, n, k, m, y, x_scales=xs, workspace=workspace)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    got = []
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got.append(y.clone())
    y.zero_()
    call()
    assert all(torch.equal(t, y) for t in got), (m, n, k)
# given codes, scales in rows of 16 bytes: 256 x 256, 256 x 128, 128 x 128, few rows
form = cl.lib().cascadia_int4_debug_fp8_gemm_form
for want, m, n, k, dtype in ((6, 3500, 3600, 1536, torch.bfloat16), (5, 1700, 3600, 1536, torch.float32),
                             (3, 2000, 1900, 1536, torch.bfloat16), (1, 9, 300, 9216, torch.float32)):
    assert form(n, k, 2, m, int(dtype == torch.float32)) == want
    record(m, n, k, dtype)
    print("recorded", m, n, k, flush=True)
"""


def test_recorded_without_any_workspace():
    r = subprocess.run([sys.executable, "-u", "-c", SCRIPT, ROOT], capture_output=True, text=True,
                       timeout=110, env=dict(os.environ))
    assert r.returncode == 0, r.stdout[-1000:] + r.stderr[-3000:]
    assert r.stdout.count("recorded") == 4
