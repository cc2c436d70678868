"""Runs the C++ test program that calls the layer norm, convolution and selective scan templates on slice views of wider tensors (two
groups, float16 and float32) and on dense copies, and compares the bits."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests", "cpp"))


@pytest.mark.gpu
def test_cpp_slice_views():
    import build as cpp_build
    exe = cpp_build.VIEWS_OUT
    if not os.path.exists(exe):
        exe = cpp_build.build_slice_views()
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    sys.stdout.write(r.stdout)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "FAILED" not in r.stdout and r.stdout.count("PASSED") == 14
