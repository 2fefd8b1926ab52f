"""The build's choices (CPU): the C library alone needs no torch, and the torch binding belongs to one
torch and one Python."""
from __future__ import annotations

import importlib.util
import subprocess

import pytest


class Compiles(Exception):
    pass


@pytest.fixture()
def build(monkeypatch):
    from dcr_b200 import build as b
    b.build()

    def run(*a, **kw):
        raise Compiles
    monkeypatch.setattr(subprocess, "run", run)
    return b


def test_the_c_library_needs_no_torch(build, monkeypatch):
    def binding(*a, **kw):
        raise AssertionError("the binding was asked for")
    monkeypatch.setattr(build, "build_torch", binding)
    find = importlib.util.find_spec
    with pytest.raises(AssertionError):
        build.build()
    assert build.build(binding=False) == build.LIB_PATH
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    assert build.build() == build.LIB_PATH


def test_a_binding_for_another_torch_is_built_again(build, monkeypatch):
    import torch
    assert build.build_torch() == build.TORCH_PATH  # up to date: nothing is compiled
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".other")
    with pytest.raises(Compiles):
        build.build_torch()
