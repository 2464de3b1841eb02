"""Status words of the serving operators, checked on the host against a
recorder in place of the CUDA runtime (tests/status_check.cpp)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.path.dirname(os.path.dirname(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")))


@pytest.mark.skipif(not shutil.which("g++") or not os.path.exists(os.path.join(CUDA, "include", "cuda_runtime.h")),
                    reason="g++ or the CUDA headers not available")
def test_a_cleared_status_word_has_been_waited_for(tmp_path):
    exe = str(tmp_path / "status_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(CUDA, "include"), "-I", os.path.join(ROOT, "include"),
                    "-I", os.path.join(ROOT, "sparse_computation_b200", "csrc"),
                    os.path.join(ROOT, "tests", "status_check.cpp"), "-o", exe], check=True, capture_output=True, text=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
