"""Routing and the 8-bit floating-point products through the C++ host API:
tests/cpp/test_cpp_fp8.cpp on the GPU, and its compilation on the CPU."""
import os
import shutil
import subprocess

import pytest
import torch

from conftest import ROOT

BIN = os.path.join(ROOT, "tests", "cpp", "_build", "test_cpp_fp8")


def test_cpp_fp8_compiles():
    if not shutil.which("g++") or not os.path.isdir("/opt/rocm/include"):
        pytest.skip("no g++ or ROCm headers")
    r = subprocess.run(["g++", "-std=c++17", "-fsyntax-only", "-Wall", "-Wextra", "-Werror",
                        "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                        "-I" + os.path.join(ROOT, "include"),
                        os.path.join(ROOT, "tests", "cpp", "test_cpp_fp8.cpp")],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-3000:]


@pytest.mark.gpu
def test_cpp_fp8():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    assert os.path.exists(BIN), f"{BIN} missing: run __graft_entry__.build()"
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=120)
    print(r.stdout[-4000:])
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    assert "checks OK" in r.stdout
