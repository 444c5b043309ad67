"""The build of the native parts: the C library needs nvcc alone, the pointwise
layers' module a torch, and the module of another torch is not taken for its own."""

from __future__ import annotations

import subprocess
import sys

import build_native
import pytest
import torch

from fast_compressai import _native


@pytest.fixture
def commands(monkeypatch):
    """The commands a build would run, which do not run."""
    run = []
    monkeypatch.setattr(subprocess, "run", lambda cmd, **kw: run.append([str(c) for c in cmd]))
    monkeypatch.setattr(build_native.os, "replace", lambda a, b: None)
    monkeypatch.setattr(build_native, "_build_lib", lambda verbose: run.append(["library"]))
    return run


def test_the_library_builds_without_torch(monkeypatch, commands):
    monkeypatch.setitem(sys.modules, "torch", None)  # importing it raises ImportError
    assert build_native.build(force=True) == build_native.LIB
    assert commands == [["library"]]


def test_what_is_built_already_is_left_alone(monkeypatch, commands):
    monkeypatch.setattr(build_native, "up_to_date", lambda: True)
    build_native.build()
    assert commands == []


def test_another_torch_gets_another_module(monkeypatch, commands):
    monkeypatch.setattr(build_native, "up_to_date", lambda: True)
    monkeypatch.setattr(torch, "__version__", "99.0.0")
    build_native.build()
    assert len(commands) == 1 and any("layers_host.cpp" in c for c in commands[0])
    monkeypatch.setattr(_native, "_host", None)
    with pytest.raises(_native.NativeLibraryError, match="not built"):
        _native.layers_host()
