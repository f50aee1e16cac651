"""The host-only test of the rule that says which shared prefixes pay."""
import os
import subprocess

import pytest

from test_planner_cpu import PKG, ROOT, _cuda_include


def test_rule_takes_the_faster_side(tmp_path):
    inc = _cuda_include()
    if inc is None:
        pytest.skip("no CUDA include directory found")
    exe = tmp_path / "prefix_rule_test"
    cmd = ["g++", "-std=c++20", "-O1", "-Wall", "-Wextra", "-I", os.path.join(ROOT, "include"), "-I", PKG, "-I", inc,
           os.path.join(ROOT, "tests", "cpp", "prefix_rule_test.cc"), "-o", str(exe)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "prefix_rule_test: ok" in r.stdout, r.stdout + r.stderr
