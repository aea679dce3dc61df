"""The build's order: the C library needs no torch, and the binding belongs to one."""
import importlib
import os
import subprocess
import sys

import pytest
import torch

import monarch_attention_b200 as mab
from monarch_attention_b200 import _lib

build = importlib.import_module("monarch_attention_b200.build")


def test_the_library_is_built_where_the_binding_cannot_be(monkeypatch):
    done = []

    def fail():
        done.append("binding")
        raise RuntimeError("no host compiler")

    monkeypatch.setattr(build, "up_to_date", lambda: False)
    monkeypatch.setattr(build, "build_library", lambda *a: done.append("library"))
    monkeypatch.setattr(build, "binding_up_to_date", lambda: False)
    monkeypatch.setattr(build, "build_binding", fail)
    with pytest.warns(UserWarning, match="no host compiler"):
        assert build.build() == build.OUT
    assert done == ["library", "binding"]


def test_a_failed_binding_leaves_no_older_one(monkeypatch, tmp_path):
    old = tmp_path / "old.so"
    old.write_bytes(b"")
    monkeypatch.setattr(build, "binding_path", lambda: str(old))
    monkeypatch.setenv("CXX", "false")
    with pytest.raises(RuntimeError, match="false failed"):
        build.build_binding()
    assert not old.exists()


def test_a_binding_for_another_torch_is_not_loaded(monkeypatch):
    path = build.binding_path()
    assert os.path.exists(path)
    monkeypatch.setattr(_lib, "_torch_binding", None)
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert build.binding_path() != path and not build.binding_up_to_date()
    with pytest.raises(RuntimeError, match=r"torch-0\.0\.1\.so"):
        _lib.load_torch_binding()
    mab.load_library()  # the library does not depend on it


def test_the_build_script_needs_no_package():
    """build.py alone, without torch, knows the library's sources and whether it is current."""
    code = ("import sys; sys.modules['torch'] = None; sys.path.insert(0, sys.argv[1]); import build; "
            "assert build.sources() and build.up_to_date() in (True, False)")
    subprocess.run([sys.executable, "-c", code, os.path.dirname(build.__file__)], check=True)
