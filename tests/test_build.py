"""CPU: what the build makes, in which order, and from what -- with the
compilers replaced by one that only creates its output."""

import importlib.util
import os

import pytest

from conftest import PKG_DIR


@pytest.fixture
def native_build(monkeypatch, tmp_path):
    """build.py with its outputs in tmp_path; .ran lists the compilers' calls."""
    spec = importlib.util.spec_from_file_location("native_build", os.path.join(PKG_DIR, "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.ran = []

    def run(cmd, verbose):
        module.ran.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w"):
            pass

    monkeypatch.setattr(module, "_run", run)
    monkeypatch.setattr(module, "nvcc_path", lambda: "nvcc")
    monkeypatch.setattr(module, "LIB", str(tmp_path / "lib.so"))
    return module


def without_torch(module, monkeypatch):
    find = importlib.util.find_spec
    monkeypatch.setattr(module.importlib.util, "find_spec",
                        lambda name, *a: None if name == "torch" else find(name, *a))


def test_the_library_needs_no_torch(native_build, monkeypatch, capsys):
    """The C library alone, from nvcc: torch is missed only by the binding."""
    without_torch(native_build, monkeypatch)
    assert native_build.build(force=True) == native_build.LIB
    assert os.path.exists(native_build.LIB)
    assert {cmd[0] for cmd in native_build.ran} == {"nvcc"}
    assert "torch" in capsys.readouterr().err


def test_the_library_comes_first(native_build, monkeypatch, tmp_path):
    """A binding that cannot be compiled leaves the library built."""
    def broken(force=False, verbose=False):
        assert os.path.exists(native_build.LIB)
        raise RuntimeError("no host compiler")

    monkeypatch.setattr(native_build, "build_binding", broken)
    with pytest.raises(RuntimeError):
        native_build.build(force=True)
    assert os.path.exists(native_build.LIB)


def test_the_binding_is_that_of_this_torch_and_python(native_build):
    """Build and package agree on the file, which names both versions."""
    import sys

    import torch
    from fast_moss_b200 import _lib

    path = _lib.binding_path()
    assert native_build.binding_path() == path and os.path.exists(path)
    assert str(torch.__version__) in path and sys.implementation.cache_tag in path


def test_another_torch_gets_a_binding_of_its_own(native_build, monkeypatch, tmp_path):
    """A binding made for one torch is neither taken for up to date nor loaded
    under another one."""
    import torch
    from fast_moss_b200 import _lib

    monkeypatch.setattr(native_build, "PACKAGE", str(tmp_path))
    native_build.build_binding()
    native_build.build_binding()
    assert len(native_build.ran) == 1
    monkeypatch.setattr(native_build, "torch_version", lambda: "99.0")
    native_build.build_binding()
    assert len(native_build.ran) == 2 and "99.0" in native_build.binding_path()

    monkeypatch.setattr(_lib, "_binding", None)
    monkeypatch.setattr(torch, "__version__", "99.0")
    with pytest.raises(ImportError, match="99.0"):
        _lib.binding()
