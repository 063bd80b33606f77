"""The host side of the batched operators on the CPU: refusals, launches,
lengths and lifetimes of gh_kv8_* and gh_sample_rows.

libgemma_hip's host code is built with g++ and a sanitizer against the
stand-ins for the HIP runtime and the other kernels (tests/cpp/hip_stub.cpp,
kernel_stub.cpp) and driven by tests/cpp/batch_ops_test.cpp, whose launchers
check what they are given."""
from __future__ import annotations

import os
import shutil
import subprocess

import numpy as np
import pytest

import gemma_hip as gh
from conftest import REPO

CSRC = REPO / "gemma.hs_amd" / "csrc"
CPP = REPO / "tests" / "cpp"


@pytest.fixture(scope="module", params=["address,undefined", "thread"])
def exe(request, tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    out = tmp_path_factory.mktemp("batch_ops") / "batch_ops_test"
    srcs = [CSRC / f for f in ("model.cpp", "gguf.cpp", "repack.cpp", "synth.cpp", "kv8.cpp", "sampling.cpp")]
    cmd = [gxx, "-std=c++17", "-g", "-O1", f"-fsanitize={request.param}", "-fno-omit-frame-pointer",
           "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{REPO / 'include'}", *map(str, srcs),
           str(CPP / "hip_stub.cpp"), str(CPP / "kernel_stub.cpp"), str(CPP / "batch_ops_test.cpp"), "-o", str(out),
           "-lpthread"]
    # kernel_stub.cpp has no launcher of the batched operators: the driver does
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    return out


@pytest.mark.parametrize("mode", ["refusals", "splits", "lifetimes"])
def test_host_side(exe, mode):
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:exitcode=23", TSAN_OPTIONS="halt_on_error=1:exitcode=24",
               UBSAN_OPTIONS="halt_on_error=1")
    env.pop("LD_PRELOAD", None)
    r = subprocess.run([str(exe), mode], capture_output=True, text=True, env=env, timeout=300)
    assert r.returncode == 0, r.stderr[-4000:]


def test_python_arguments():
    """What the Python side refuses before any call."""
    assert gh.SAMPLING.itemsize == 20
    r = gh.sampling(3, 0.7, top_k=[1, 2, 3])
    assert r["top_p"].tolist() == [1, 1, 1] and r["top_k"].tolist() == [1, 2, 3] and r["min_p"].tolist() == [0, 0, 0]
    with pytest.raises(ValueError):
        gh.sample_rows(None, 0, 10, np.zeros((2, 2), gh.SAMPLING))
    with pytest.raises(ValueError):
        gh.sample_rows(None, 0, 10, np.zeros(2, np.float32))
    with pytest.raises(ValueError):
        gh._ints([0, 1], [1])
    with pytest.raises(ValueError):
        gh._ints([[0]], [[1]])
