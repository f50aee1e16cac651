"""The host-only test of when the work lists of the long-context decode calls are made."""
import os
import subprocess

import pytest

from test_planner_cpu import PKG, ROOT, _cuda_include


def test_layers_that_come_again_plan_again(tmp_path):
    inc = _cuda_include()
    if inc is None:
        pytest.skip("no CUDA include directory found")
    exe = tmp_path / "step_layers_test"
    cmd = ["g++", "-std=c++20", "-O1", "-Wall", "-Wextra", "-I", os.path.join(ROOT, "include"), "-I", PKG, "-I", inc,
           os.path.join(ROOT, "tests", "cpp", "step_layers_test.cc"), "-o", str(exe)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "step_layers_test: ok" in r.stdout, r.stdout + r.stderr
