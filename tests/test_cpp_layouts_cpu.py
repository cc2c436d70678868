"""The layouts that the C++ templates of layer norm, convolution and selective scan take and refuse: tests/cpp/layout_refusals.cpp calls
each with tensors that have no memory, so nothing runs on a GPU. A refused layout ends with the template's own message; one that is
taken gets as far as the first allocation or the library's check for null pointers."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests", "cpp"))

TAKEN = ["scan", "scan gradient", "scan rows of groups", "scan one group of wider rows", "scan channels of wider rows", "step", "step rows of groups",
         "step one group of wider rows", "norm", "norm gradient", "norm of wider rows", "norm of one row",
         "conv", "conv gradient", "conv of wider rows"]
REFUSED = {
    "scan B of sliced states": "not evenly spaced", "scan C of sliced states": "not evenly spaced",
    "scan gradient C of sliced states": "not evenly spaced", "scan B states apart": "not evenly spaced", "scan channels apart": "not evenly spaced",
    "scan gradient dy channels apart": "dy does not match x", "step B of sliced states": "rows are not dense", "step C of sliced states": "rows are not dense",
    "step channels apart": "rows are not dense",
    "norm of cut rows": "evenly spaced", "norm columns apart": "evenly spaced", "norm gradient of cut rows": "evenly spaced",
    "norm gradient of cut dy": "evenly spaced",
    "conv sliced w": "dense", "conv channels apart": "dense", "conv gradient sliced w": "dense", "conv gradient channels apart": "dense",
    "scan sliced A": "dense", "scan sliced initial states": "dense", "scan gradient sliced dfinal states": "dense", "step sliced A": "dense",
    "step sliced state": "dense",
}


@pytest.fixture(scope="module")
def program():
    import build as cpp_build
    return cpp_build.build_layout_refusals()  # always: the headers are part of it


def run(program, case):
    r = subprocess.run([program, case], capture_output=True, text=True, timeout=60, env={**os.environ, "CUDA_VISIBLE_DEVICES": ""})
    assert r.returncode == 1, (case, r.returncode, r.stdout + r.stderr)
    return r.stdout


@pytest.mark.parametrize("case", TAKEN)
def test_taken(program, case):
    out = run(program, case)
    assert "code: " in out or "null pointer" in out, out


@pytest.mark.parametrize("case", sorted(REFUSED))
def test_refused(program, case):
    assert REFUSED[case] in run(program, case)
