"""Waits inside the LM head's tensor-memory kernel that run out: the launch ends, says so, and leaves the device as it was (tests/late_head.cu)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu


def test_waits_that_run_out(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc on this machine")
    exe = str(tmp_path / "late_head")
    csrc = os.path.join(ROOT, "ferro_b200", "csrc")
    r = subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-t", "3", "-include", os.path.join(ROOT, "tests", "late_head.cuh"),
                        "-o", exe, os.path.join(ROOT, "tests", "late_head.cu"), os.path.join(csrc, "fsb_head.cu"), os.path.join(csrc, "fsb_head_many.cu")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    told0, right0, told1, right1 = map(int, r.stdout.split())
    assert min(told0, told1) >= 5 and min(right0, right1) >= 5, r.stdout
