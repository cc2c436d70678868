"""build() of __graft_entry__ compiles the product whatever the test tree beside it holds: the C++ test programs are built where that
tree has them, and a tree without one of them (an older one, or none at all) does not stop the build. No GPU, no compiler."""
import os
import sys
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

import __graft_entry__ as entry  # noqa: E402
from anygpu_b200 import build as product, capi  # noqa: E402
from oracle import oracle  # noqa: E402


@pytest.mark.parametrize("programs", [(), ("build",), ("build", "build_sft_dump"), ("build", "build_sft_dump", "build_selective_scan_layer")])
def test_build_takes_any_test_tree(monkeypatch, programs):
    done = []
    monkeypatch.setattr(product, "build", lambda *a, **k: done.append("library"))
    monkeypatch.setattr(oracle, "build", lambda *a, **k: done.append("oracle"))
    monkeypatch.setattr(capi, "load", lambda: done.append("load"))
    monkeypatch.setattr(sys, "path", list(sys.path))
    tree = types.ModuleType("build")
    for name in programs:
        setattr(tree, name, lambda name=name: done.append(name))
    monkeypatch.setitem(sys.modules, "build", tree)
    entry.build()
    assert done[:3] == ["library", "oracle", "load"]
    assert done[3:] == [name for name in programs if name != "build_sft_dump"]


def test_build_without_a_test_tree(monkeypatch):
    done = []
    monkeypatch.setattr(product, "build", lambda *a, **k: done.append("library"))
    monkeypatch.setattr(oracle, "build", lambda *a, **k: done.append("oracle"))
    monkeypatch.setattr(capi, "load", lambda: done.append("load"))
    monkeypatch.setattr(sys, "path", list(sys.path))
    monkeypatch.setattr(entry, "ROOT", os.path.join(ROOT, "nowhere"))
    monkeypatch.delitem(sys.modules, "build", raising=False)
    entry.build()
    assert done == ["library", "oracle", "load"] and not any("nowhere" in p for p in sys.path)
