"""The overlap checks of the losses (host code, no device), built with
AddressSanitizer and UndefinedBehaviorSanitizer."""

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_overlaps_against_sets_of_bytes(tmp_path):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "learn_ranges")
    build = subprocess.run(
        [gxx, "-std=c++17", "-O1", "-g", "-Wall", "-Wextra", "-fno-omit-frame-pointer",
         "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
         "-I" + os.path.join(ROOT, "metalfish_amd", "csrc", "hip"),
         os.path.join(ROOT, "tests", "native", "learn_ranges_test.cpp"), "-o", exe],
        capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
    assert "learn ranges ok" in run.stdout
