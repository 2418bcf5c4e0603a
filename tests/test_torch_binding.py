"""Which compiled way from torch tensors to the library is built and loaded, without a GPU."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from teamredbench_b200 import _native, build  # noqa: E402


@pytest.fixture
def nothing_else_stale(monkeypatch):
    """build() has only the binding to look at; the commands that it runs are listed, not run."""
    commands = []
    monkeypatch.setattr(build, "find_nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    real = build._stale
    monkeypatch.setattr(build, "_stale", lambda target, deps: "torch" in target.name and real(target, deps))
    monkeypatch.setattr(build, "_run", lambda cmd, verbose: commands.append(cmd) or "")
    return commands


def _built():
    if _native.load_torch_binding() is None:
        pytest.skip("not built (python -m teamredbench_b200.build)")


def test_a_binding_of_another_torch_is_not_loaded(monkeypatch):
    _built()
    monkeypatch.setattr(torch, "__version__", "1.0.0+other")
    assert _native.load_torch_binding() is None


def test_a_binding_of_another_python_is_not_loaded(monkeypatch):
    _built()
    real = _native.sysconfig.get_config_var
    monkeypatch.setattr(_native.sysconfig, "get_config_var", lambda name: "cpython-30" if name == "SOABI" else real(name))
    assert _native.load_torch_binding() is None


def test_another_torch_gets_a_binding_of_its_own(monkeypatch, nothing_else_stale):
    _built()
    build.build()
    assert nothing_else_stale == []
    monkeypatch.setattr(torch, "__version__", "1.0.0+other")
    build.build()
    (command,) = nothing_else_stale
    target = command[command.index("-o") + 1]
    assert target == str(_native.torch_binding_path()) and "1.0.0+other" in target


@pytest.fixture
def elsewhere(monkeypatch, tmp_path, nothing_else_stale):
    """The binding's file is another one, which an older source has left."""
    monkeypatch.setattr(_native, "LIB_DIR", tmp_path)
    left = _native.torch_binding_path()
    left.touch()
    monkeypatch.setattr(build, "_stale", lambda target, deps: "torch" in target.name)
    return left


@pytest.mark.parametrize("error", [RuntimeError("Python.h: No such file"), ImportError("libc10"), OSError("libcudart")])
@pytest.mark.parametrize("where", ["_run", "_torch_binding_command"])
def test_a_binding_that_cannot_be_built_is_a_warning(monkeypatch, elsewhere, where, error):
    """The library and the executables are there, and the front ends work without the binding."""
    def fail(*_):
        raise error

    monkeypatch.setattr(build, where, fail)
    with pytest.warns(RuntimeWarning, match=str(error)):
        assert build.build() == build.LIBRARY
    assert not elsewhere.exists()  # made for another header, maybe
    monkeypatch.setattr(_native, "load", lambda: None)
    assert _native.load_torch_binding() is None


def test_a_compiler_that_fails_is_a_warning(monkeypatch, elsewhere):
    monkeypatch.undo()
    monkeypatch.setenv("CXX", "/bin/false")
    monkeypatch.setattr(_native, "LIB_DIR", elsewhere.parent)
    monkeypatch.setattr(build, "find_nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    monkeypatch.setattr(build, "_stale", lambda target, deps: "torch" in target.name)
    with pytest.warns(RuntimeWarning, match="command failed"):
        build.build()
    assert not elsewhere.exists()


def test_a_torch_without_cuda_needs_no_binding(monkeypatch, elsewhere, nothing_else_stale, recwarn):
    monkeypatch.setattr(torch.version, "cuda", None)
    assert build.build() == build.LIBRARY
    assert nothing_else_stale == [] and not recwarn.list
