"""Plans made by hand in the C++ mirror: it compiles (CPU check) and refuses tables that do not fit (GPU, for the buffers)."""
import os
import shutil
import subprocess

import pytest

from ferro_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "cpp", "layer_plans_test.cpp")
BIN = os.path.join(ROOT, "ferro_b200", "lib", "layer_plans_test")


def compile_test():
    build.build()
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    lib_dir = os.path.join(ROOT, "ferro_b200", "lib")
    subprocess.run([nvcc, "-std=c++17", "-O1", "-x", "cu", "-gencode", "arch=compute_100a,code=sm_100a", SRC, "-o", BIN,
                    "-L", lib_dir, "-lferro_b200", "-cudart", "shared", "-Xlinker", f"-rpath={lib_dir}"], check=True)
    return BIN


def test_cpp_layer_plans_compile_and_link():
    assert os.path.exists(compile_test())


@pytest.mark.gpu
def test_cpp_plans_that_do_not_fit_are_refused():
    r = subprocess.run([compile_test()], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "layer_plans_test ok" in r.stdout
