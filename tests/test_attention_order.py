"""The order of workgroups of causal attention (host code, no device)."""

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_tiles_of_causal_rows(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    exe = str(tmp_path / "attention_order")
    build = subprocess.run(
        [hipcc, "--offload-arch=gfx950", "--offload-host-only", "-std=c++17", "-O1", "-x", "hip",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-I" + os.path.join(ROOT, "metalfish_amd", "csrc", "hip"),
         os.path.join(ROOT, "tests", "native", "attention_order_test.cpp"), "-o", exe],
        capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
    assert "attention order ok" in run.stdout
