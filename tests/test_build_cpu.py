"""What the build does where parts of it cannot be built."""

import stat

import pytest

from neuralzip_b200 import build


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
