"""The library's Makefile: what the default target needs, and when the Python
module is built again.  Compilers are stand-ins; nothing is compiled."""
import os
import shutil
import subprocess
import sys

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "minicpm-v-4.6-orangepi_b200")


@pytest.fixture
def tree(tmp_path):
    (tmp_path / "csrc").mkdir()
    (tmp_path / "mcv_b200").mkdir()
    shutil.copy(os.path.join(PKG, "Makefile"), tmp_path)
    (tmp_path / "csrc" / "tensors.cpp").write_text("")
    return tmp_path


def make(tree, *args):
    # the stand-in writes the file behind -o
    write = "sh -c 'while [ $$# -gt 0 ]; do [ \"$$1\" = -o ] && echo x > $$2; shift; done' --"
    r = subprocess.run(["make", "-C", str(tree), f"PYTHON={sys.executable}", f"CXX={write}", f"NVCC={write}", *args],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_library_alone_without_torch(tree):
    out = make(tree, "PYTHON=/nonexistent/python", "NCCL_HOME=/nonexistent")
    assert (tree / "libmcv_b200.so").exists() and not (tree / "mcv_b200" / "_tensors.so").exists()
    assert "tensors.cpp" not in out


def test_module_follows_torch_and_python(tree):
    assert "tensors.cpp" in make(tree, "TORCH_ID=2.0 cpython-312")
    assert (tree / "mcv_b200" / "_tensors.so").exists()
    assert "tensors.cpp" not in make(tree, "TORCH_ID=2.0 cpython-312")
    for changed in ("TORCH_ID=2.1 cpython-312", "TORCH_ID=2.1 cpython-313"):
        os.utime(tree / "mcv_b200" / "_tensors.so", (1, 1))
        os.utime(tree / "_build" / "python_torch", (1, 1))
        os.utime(tree / "csrc" / "tensors.cpp", (1, 1))
        assert "tensors.cpp" in make(tree, changed)
        assert "tensors.cpp" not in make(tree, changed)
