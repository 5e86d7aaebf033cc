"""Finding the compiled parts."""

import sys

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
