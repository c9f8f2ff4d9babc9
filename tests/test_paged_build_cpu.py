"""The library is built without Python's or torch's headers, and the paged memory's calls do without their native module."""
import sys
import types
import warnings

import pytest
import torch

import sarbon_b200
from sarbon_b200 import _lib, build_lib, paged_ops

needs_library = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="not built")


def test_the_library_is_built_without_the_module(monkeypatch, tmp_path):
    stale, other = tmp_path / "_paged_calls.here.so", tmp_path / "_paged_calls.so"
    for f in (stale, other):
        f.write_bytes(b"")
    done = []

    def no_headers(force, verbose):
        done.append("module")
        raise RuntimeError("Python.h: No such file or directory")

    monkeypatch.setattr(build_lib, "PKG", tmp_path)
    monkeypatch.setattr(build_lib, "CALLS_LIB", stale)
    monkeypatch.setattr(build_lib, "build_library", lambda *a: done.append("library") or "the library")
    monkeypatch.setattr(build_lib, "build_calls", no_headers)
    with pytest.warns(RuntimeWarning, match="Python.h"):
        assert build_lib.build() == "the library"
    assert done == ["library", "module"]
    assert not stale.exists() and not other.exists()  # neither could be trusted to fit the library


def test_the_module_is_built_again_for_another_torch(monkeypatch, tmp_path):
    runs = []

    def compiler(what, cmd):
        runs.append(cmd)
        open(cmd[cmd.index("-o") + 1], "wb").close()

    for name, path in dict(OBJ=tmp_path / "obj", CALLS_LIB=tmp_path / "_paged_calls.here.so", CALLS_FOR=tmp_path / "obj" / "for.txt").items():
        monkeypatch.setattr(build_lib, name, path)
    monkeypatch.setattr(build_lib, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    monkeypatch.setattr(build_lib, "_run", compiler)
    build_lib.build_calls()
    build_lib.build_calls()
    assert len(runs) == 1 and any(torch.__version__ in x for x in runs[0])
    monkeypatch.setattr(torch, "__version__", "9.9.9+else")
    build_lib.build_calls()
    assert len(runs) == 2 and any("9.9.9+else" in x for x in runs[1])


@needs_library
@pytest.mark.parametrize("module", [None, types.SimpleNamespace(built_for="1.0.0")])
def test_calls_without_the_module(monkeypatch, module):
    monkeypatch.setattr(paged_ops, "_native", None)
    monkeypatch.delattr(sarbon_b200, "_paged_calls", raising=False)
    monkeypatch.setitem(sys.modules, "sarbon_b200._paged_calls", module)
    with pytest.warns(RuntimeWarning, match="host"):
        side = paged_ops._load()
    assert side.attend(1, 2) is None and side.append() is None and side.cut(3) is None
    assert paged_ops._native is side  # and said once


@needs_library
def test_the_module_that_was_built_is_used(monkeypatch):
    if not build_lib.CALLS_LIB.exists():
        pytest.skip("not built")
    monkeypatch.setattr(paged_ops, "_native", None)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        side = paged_ops._load()
    assert side.built_for == torch.__version__ and side.__file__ == str(build_lib.CALLS_LIB)
