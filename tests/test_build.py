"""Building and finding the compiled parts, with the compilers faked."""

import subprocess
import sys
from pathlib import Path

import pytest
import torch

from ninetoothed_b200 import _build, _lib


@pytest.fixture
def unbound(monkeypatch):
    monkeypatch.setattr(_lib, "_binding", None)


def test_binding_is_taken_only_by_the_torch_it_was_built_for(monkeypatch, unbound):
    assert not _build.binding_is_stale()
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", torch.__version__ + ".other")
        assert _build.binding_is_stale() and _build.is_stale()
        assert _lib.binding() is None
    _lib._binding = None
    assert _lib.binding() is not None


def test_binding_is_taken_only_by_the_python_it_was_built_for(monkeypatch, unbound):
    monkeypatch.setattr(sys.implementation, "cache_tag", "cpython-00")
    assert _build.binding_is_stale()
    assert _lib.binding() is None


@pytest.mark.parametrize("force", (False, True))
def test_library_is_built_where_the_binding_cannot_be(force, monkeypatch, tmp_path):
    ran = []

    def run(command, check):
        ran.append(command[0])
        if command[0] == "g++":
            raise subprocess.CalledProcessError(1, command)
        Path(command[command.index("-o") + 1]).write_bytes(b"library")

    monkeypatch.setattr(_build, "PACKAGE_DIR", tmp_path)
    monkeypatch.setattr(_build, "LIBRARY", tmp_path / "libnt_b200.so")
    monkeypatch.setattr(_build, "find_nvcc", lambda: "nvcc")
    monkeypatch.setattr(_build.subprocess, "run", run)
    with pytest.warns(UserWarning, match="binding"):
        assert _build.build(force=force) == tmp_path / "libnt_b200.so"
    assert (tmp_path / "libnt_b200.so").read_bytes() == b"library" and ran == ["nvcc", "g++"]
    assert [p.name for p in tmp_path.iterdir()] == ["libnt_b200.so"]


def test_missing_compiler_of_the_binding(monkeypatch, tmp_path):
    def run(command, check):
        if command[0] == "g++":
            raise FileNotFoundError("g++")
        Path(command[command.index("-o") + 1]).write_bytes(b"library")

    monkeypatch.setattr(_build, "PACKAGE_DIR", tmp_path)
    monkeypatch.setattr(_build, "LIBRARY", tmp_path / "libnt_b200.so")
    monkeypatch.setattr(_build, "find_nvcc", lambda: "nvcc")
    monkeypatch.setattr(_build.subprocess, "run", run)
    with pytest.warns(UserWarning, match="binding"):
        _build.build()
    assert (tmp_path / "libnt_b200.so").is_file()
