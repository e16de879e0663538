"""What the build does where parts of it cannot be built."""

import importlib.machinery
import importlib.util
import stat
import types

import pytest
import torch

from neuralzip_b200 import build
from neuralzip_b200.gpu import paged


@pytest.fixture
def elsewhere(tmp_path, monkeypatch):
    """Outputs in a folder of the test's, and a compiler for the library that only leaves a file."""
    nvcc = tmp_path / "nvcc"
    nvcc.write_text('#!/bin/sh\nwhile [ "$1" != -o ]; do shift; done\necho library > "$2"\n')
    nvcc.chmod(nvcc.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setattr(build, "OUTPUT", tmp_path / "lib" / "library.so")
    monkeypatch.setattr(build, "nvcc", lambda: str(nvcc))
    return tmp_path / "lib"


@pytest.mark.parametrize("compiler", ["false", "/nonexistent/g++"])
def test_the_library_does_not_need_the_torch_calls(elsewhere, monkeypatch, compiler):
    monkeypatch.setenv("CXX", compiler)
    for force in (False, True):
        if force:  # left by an older source: not to be used with this library
            build.torch_calls().write_text("old")
        with pytest.warns(UserWarning, match="was not built"):
            assert build.build(force=force) == elsewhere / "library.so"
        assert (elsewhere / "library.so").read_text() == "library\n"
        assert [path.name for path in elsewhere.iterdir()] == ["library.so"]


def test_torch_calls_of_another_torch_are_not_loaded(monkeypatch):
    """A module that was built against another torch or Python may load all the same, and misread their objects."""
    module = types.SimpleNamespace(bind=lambda *_: None)
    monkeypatch.setattr(paged, "_calls", None)
    monkeypatch.setattr(importlib.util, "module_from_spec", lambda spec: module)
    loaded = []

    def load(self, module):
        loaded.append(self.path)
        if self.path != str(build.torch_calls()) or not build.torch_calls().exists():
            raise ImportError(self.path)

    monkeypatch.setattr(importlib.machinery.ExtensionFileLoader, "exec_module", load)
    if not build.torch_calls().exists():
        pytest.skip("The torch calls were not built.")
    paged._load_calls.__wrapped__()
    assert paged._calls is module
    mine = build.torch_calls()
    for name, value in (("torch", "0.1.2"), ("soabi", "cpython-30")):
        with monkeypatch.context() as change:
            if name == "torch":
                change.setattr(torch, "__version__", value)
            else:
                change.setattr(build.sysconfig, "get_config_var", lambda _: value)
            change.setattr(paged, "_calls", None)
            paged._load_calls.__wrapped__()
            assert paged._calls is None and loaded[-1] != str(mine)
            assert build._stale(build.torch_calls(), [])  # and the build makes one for this torch
