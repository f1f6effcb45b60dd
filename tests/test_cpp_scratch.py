"""Scratch of the C++ mirror after a request that could not be met."""
import os
import shutil
import subprocess

import pytest

from ferro_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "cpp", "scratch_test.cpp")
BIN = os.path.join(ROOT, "ferro_b200", "lib", "scratch_test")


def compile_test():
    build.build()
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    lib_dir = os.path.join(ROOT, "ferro_b200", "lib")
    subprocess.run([nvcc, "-std=c++17", "-O1", "-x", "cu", "-gencode", "arch=compute_100a,code=sm_100a", SRC, "-o", BIN,
                    "-L", lib_dir, "-lferro_b200", "-cudart", "shared", "-Xlinker", f"-rpath={lib_dir}"], check=True)
    return BIN


def test_cpp_scratch_compile_and_link():
    assert os.path.exists(compile_test())


@pytest.mark.gpu
def test_cpp_scratch_that_could_not_be_had_is_forgotten():
    r = subprocess.run([compile_test()], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "scratch_test ok" in r.stdout
