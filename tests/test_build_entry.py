"""CPU: build() compiles, whatever is there; smoke() and the tests load what is built."""
import importlib
import os

from conftest import ROOT, load_pkg


def test_build_compiles_what_is_built_already(monkeypatch):
    load_pkg()
    entry = importlib.import_module("__graft_entry__")
    calls = []
    monkeypatch.setattr(entry.subprocess, "check_call", calls.append)
    entry.build()
    assert [os.path.relpath(c[c.index("-C") + 1], ROOT) for c in calls] == [os.path.join("semantic-segmentation_amd", "csrc"), "oracle"]
    assert all(c[0] == "make" and "-B" in c for c in calls)


def test_the_library_depends_on_all_of_its_sources():
    """Every source and header of csrc/ is named in its Makefile."""
    csrc = os.path.join(ROOT, "semantic-segmentation_amd", "csrc")
    text = open(os.path.join(csrc, "Makefile")).read()
    missing = [f for f in sorted(os.listdir(csrc)) if f.endswith((".hip", ".h", ".cpp")) and f not in text]
    assert not missing
