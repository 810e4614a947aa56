"""CPU test of the sampling kernel's layout of rows of every vocabulary."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_parts_cover_the_row_and_fit_the_step_sums(tmp_path):
    exe = tmp_path / "sample_plan_check"
    src = os.path.join(ROOT, "tests", "native", "sample_plan_check.cpp")
    inc = os.path.join(ROOT, "walsh_research_b200", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O2", "-I" + inc, src, "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "sample_plan ok" in r.stdout
