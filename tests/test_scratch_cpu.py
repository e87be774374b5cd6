"""CPU tests of a context's scratch: scratch.cpp runs it against a stand-in for the CUDA runtime."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CUDA = os.path.dirname(os.path.dirname(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")))


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("scratch") / "scratch")
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", os.path.join(CUDA, "include"), "-o", out, os.path.join(HERE, "scratch.cpp")], check=True)
    return out


@pytest.mark.parametrize("scenario", ["grows", "out of memory", "out of memory for both", "out of memory and kept for a graph", "out of memory for counters", "in a capture", "kept for a graph", "kept only if captured", "rising little by little",
                                      "half as much again does not fit", "held by another thread",
                                      "no wait for the device during a capture"])
def test_scenario(program, scenario):
    r = subprocess.run([program, scenario], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
