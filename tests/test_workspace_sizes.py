"""Workspace sizes asked for with sizes past 32 bits, negative ones, or none: refused as
arguments, not cut off to 32 bits (Python and C++)."""
import os
import subprocess

import pytest
import torch

from conftest import ROOT

BIN = os.path.join(ROOT, "tests", "cpp", "_build", "test_cpp_sizes")
PAST = 1 << 32


@pytest.fixture(scope="module")
def cl():
    import cascadia_amd

    return cascadia_amd


class Layer:
    """Stands in for experts or adapters: their dimensions alone matter."""

    def __init__(self, struct):
        import ctypes

        self._set, self._ref = struct, ctypes.byref(struct)

    def _struct(self):
        return self._set


def sizes(cl):
    lib = cl._lib
    moe = Layer(lib.MoeLayer(256, 128, 32, cl.SCALE_BF16, cl.TILING_CRATE, 4, 256, 1 << 20))
    fp8 = Layer(lib.Fp8MoeLayer(256, 128, 4, 256, 256, 256, 256, 0))
    set_ = Layer(lib.AdapterSet(64, 48, 16, 4, 256, 256, 0, 0))
    return [  # (call, sizes that it takes)
        (lambda n: cl.sort_tokens_workspace_bytes(n, 8, 384), 9000),
        (lambda n: cl.sort_tokens_workspace_bytes(9000, n, 384), 8),
        (lambda n: cl.sort_tokens_workspace_bytes(9000, 8, n), 384),
        (lambda n: cl.adapters_workspace_bytes(set_, n), 40),
        (lambda n: cl.moe_workspace_bytes(moe, 2, n), 40),
        (lambda n: cl.moe_workspace_bytes(moe, n, 40), 2),
        (lambda n: cl.fp8_moe_workspace_bytes(fp8, 2, n), 40),
        (lambda n: cl.fp8_moe_workspace_bytes(fp8, n, 40), 2),
        (lambda n: cl.fp8_gemm_workspace_bytes(n, 256, 400), 128),
        (lambda n: cl.fp8_gemm_workspace_bytes(128, n, 400), 256),
        (lambda n: cl.fp8_gemm_workspace_bytes(128, 256, n), 400),
        (lambda n: cl.gemm_workspace_bytes(256, 512, n, True), 300),
        (lambda n: cl.ffn_workspace_bytes(256, 128, n), 40),
        (lambda n: cl.ffn_sparse_workspace_bytes(256, 128, n), 40),
        (lambda n: cl.ffn_sparse_axpy_workspace_bytes(256, 128, n), 40),
    ]


@pytest.mark.parametrize("which", range(15))
def test_python_sizes(cl, which):
    call, n = sizes(cl)[which]
    size = call(n)
    assert isinstance(size, int) and size >= 0
    for bad in (PAST + n, -PAST + n, PAST, -1, -n):
        with pytest.raises(ValueError):
            call(bad)
    with pytest.raises(TypeError):
        call(float(n))


def run(*args):
    if not os.path.exists(BIN):
        pytest.skip(f"{BIN} is not built")
    r = subprocess.run([BIN, *args], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    assert "checks OK" in r.stdout


def test_cpp_sizes():
    run()


@pytest.mark.gpu
def test_cpp_sizes_of_layers():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    run("device")
