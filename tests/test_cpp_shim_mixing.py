"""The token-mixing calls of the C++ shim (include/mcv_ops.hpp): compiled and
refused on the host, and a tiny layer step on a GPU (tests/shim_mixing.cpp)."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT

PKG = os.path.join(ROOT, "minicpm-v-4.6-orangepi_b200")
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


def _build(tmp_path):
    if shutil.which("g++") is None or not os.path.exists(os.path.join(CUDA, "include", "cuda_runtime_api.h")):
        pytest.skip("g++ or the CUDA headers are missing")
    exe = str(tmp_path / "shim_mixing")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-I",
                    os.path.join(CUDA, "include"), os.path.join(ROOT, "tests", "shim_mixing.cpp"), "-o", exe, "-L", PKG,
                    "-lmcv_b200", f"-Wl,-rpath,{PKG}", "-L", os.path.join(CUDA, "lib64"), "-lcudart",
                    f"-Wl,-rpath,{os.path.join(CUDA, 'lib64')}"], check=True, capture_output=True, text=True, timeout=300)
    return exe


def test_shim_mixing_refusals(tmp_path):
    out = subprocess.run([_build(tmp_path)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and "mixing ok" in out.stdout, out.stdout + out.stderr


@pytest.mark.gpu
def test_shim_mixing_on_gpu(cuda, tmp_path):
    out = subprocess.run([_build(tmp_path), "gpu"], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and "mixing ok" in out.stdout, out.stdout + out.stderr
