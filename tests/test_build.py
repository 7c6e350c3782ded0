"""The build where not everything is there."""

from __future__ import annotations

import importlib.util
import shutil
from pathlib import Path

import pytest

from conftest import PKG


@pytest.fixture
def build(tmp_path, monkeypatch):
    """build.py, with one source and its results in a directory of their own."""
    spec = importlib.util.spec_from_file_location("vmoe_build_under_test", PKG / "build.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    try:
        module.hipcc()
    except RuntimeError:
        pytest.skip("needs hipcc")
    monkeypatch.setattr(module, "SOURCES", ["capi.hip"])
    monkeypatch.setattr(module, "OBJ", tmp_path / "obj")
    monkeypatch.setattr(module, "OUT", tmp_path / "libvmoe.so")
    monkeypatch.setattr(module, "DENSE", tmp_path / "_dense.so")
    module.DENSE.write_bytes(b"of an earlier build")
    return module


def no_torch(build, monkeypatch, tmp_path):
    find = importlib.util.find_spec
    monkeypatch.setattr(build.importlib.util, "find_spec",
                        lambda name, *a: None if name == "torch" else find(name, *a))


def no_headers(build, monkeypatch, tmp_path):
    monkeypatch.setattr(build, "_torch_dir", lambda: tmp_path)


def no_compiler(build, monkeypatch, tmp_path):
    monkeypatch.setenv("CXX", "no-such-compiler")


@pytest.mark.parametrize("without", [no_torch, no_headers, no_compiler])
def test_library_without_the_extension_module(without, build, monkeypatch, tmp_path, capsys):
    """libvmoe.so, which C callers use, needs neither torch nor a host compiler. The
    extension module of an earlier build goes: it may not fit."""
    without(build, monkeypatch, tmp_path)
    assert build.build() == build.OUT and build.OUT.stat().st_size > 0
    assert not build.DENSE.exists()
    assert "_dense.so is not built" in capsys.readouterr().err


def test_errors_of_the_extension_module_are_errors(build, monkeypatch, tmp_path):
    if shutil.which("g++") is None or importlib.util.find_spec("torch") is None:
        pytest.skip("needs g++ and torch")
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    (csrc / "dense_torch.cpp").write_text("#error here\n")
    monkeypatch.setattr(build, "CSRC", Path(csrc))
    with pytest.raises(RuntimeError, match="dense_torch.cpp"):
        build._compile_dense()
