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
