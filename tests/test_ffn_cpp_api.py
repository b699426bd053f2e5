"""Compiles and runs tests/cpp/ffn_api_test.cpp against libfelix_b200.so: the
feed-forward operators as C++ callers use them."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


@pytest.fixture(scope="module")
def binary(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("cpp") / "ffn_api_test")
    cmd = ["g++", "-std=c++20", "-O1", os.path.join(ROOT, "tests", "cpp", "ffn_api_test.cpp"),
           f"-I{ROOT}/include", f"-I{CUDA}/include", f"-L{ROOT}/sion_b200", "-lfelix_b200",
           f"-Wl,-rpath,{ROOT}/sion_b200", f"-L{CUDA}/lib64", "-lcudart", "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return out


def _run(binary, *args):
    r = subprocess.run([binary, *args], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "all checks passed" in r.stdout, r.stdout + r.stderr


def test_ffn_cpp_api_without_a_device(binary):
    _run(binary)


@pytest.mark.gpu
def test_ffn_cpp_api_gpu(binary):
    _run(binary, "gpu")
