"""The in-tree build's decisions -- what is compiled, what is linked, what is left alone -- with a stand-in for hipcc (no GPU, no compiler)."""
import importlib.util
import os
import stat

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """(module, calls): build_ext over two small sources in a folder of its own; calls() gives the compiler's lines since the last time."""
    spec = importlib.util.spec_from_file_location("build_ext_under_test", os.path.join(REPO, "u-rnn_amd", "build_ext.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    log, cc = tmp_path / "calls", tmp_path / "cc"
    cc.write_text('#!/bin/sh\necho "$@" >> %s\nwhile [ $# -gt 1 ]; do if [ "$1" = -o ]; then echo made > "$2"; fi; shift; done\n' % log)
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    for name in ("a.hip", "b.hip", "common.h"):
        (tmp_path / name).write_text("//")
        os.utime(tmp_path / name, (1e9, 1e9))
    monkeypatch.setenv("HIPCC", str(cc))
    monkeypatch.setattr(mod, "CSRC", str(tmp_path))
    monkeypatch.setattr(mod, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(mod, "SOURCES", ["a.hip", "b.hip"])
    monkeypatch.setattr(mod, "HEADERS", ["common.h"])

    def calls():
        lines = log.read_text().splitlines() if log.exists() else []
        log.unlink(missing_ok=True)
        return sorted("link" if "-shared" in ln else next(w for w in ln.split() if w.endswith(".hip")).rsplit("/", 1)[1] for ln in lines)
    return mod, calls, tmp_path


def test_a_current_tree_needs_no_compiler(tree, monkeypatch):
    mod, calls, d = tree
    assert mod.build() == str(d / "lib.so") and calls() == ["a.hip", "b.hip", "link"]
    before = os.stat(d / "lib.so").st_mtime_ns
    assert mod.build() == str(d / "lib.so") and calls() == [] and os.stat(d / "lib.so").st_mtime_ns == before
    (d / "cc").unlink()                                        # a machine without one
    assert mod.build() == str(d / "lib.so")


def test_what_changed_is_built_and_linked(tree, monkeypatch):
    mod, calls, d = tree
    mod.build()
    calls()
    os.utime(d / "b.hip")                                      # a newer source
    os.utime(d / "a.o", (1.1e9, 1.1e9))
    os.utime(d / "b.o", (1.1e9, 1.1e9))
    mod.build()
    assert calls() == ["b.hip", "link"]
    os.utime(d / "common.h")                                   # a newer header
    for f in ("a.o", "b.o"):
        os.utime(d / f, (1.2e9, 1.2e9))
    mod.build()
    assert calls() == ["a.hip", "b.hip", "link"]
    monkeypatch.setattr(mod, "NO_PACKED_F32", (*mod.NO_PACKED_F32, "-DMORE"))      # another command line
    mod.build()
    assert calls() == ["a.hip", "b.hip", "link"]
    (d / "lib.so").unlink()                                    # no library
    mod.build()
    assert calls() == ["link"]
    os.utime(d / "lib.so", (1.1e9, 1.1e9))                     # one older than its objects
    mod.build()
    assert calls() == ["link"]
    monkeypatch.setattr(mod, "SOURCES", ["a.hip"])             # a unit less: the same objects, another library
    mod.build()
    assert calls() == ["link"]
    mod.build()
    assert calls() == []
    mod.build(force=True)
    assert calls() == ["a.hip", "link"]
