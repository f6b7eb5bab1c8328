"""The build of the torch-facing module, with the compiler replaced."""

from __future__ import annotations

import os
import subprocess
import sys
from types import SimpleNamespace

import pytest
import torch

from kernel_mcts_b200 import _native, build


@pytest.fixture
def compiled(monkeypatch, tmp_path):
    """A build that writes to tmp_path and only records the commands; returns them."""
    commands = []

    def run(command):
        commands.append(command)
        build.TORCH_CALLS.write_bytes(b"")

    monkeypatch.setattr(build, "TORCH_CALLS", tmp_path / "calls.so")
    monkeypatch.setattr(build, "TORCH_CALLS_BUILT_FOR", tmp_path / "calls.built_for")
    monkeypatch.setattr(build, "build_library", lambda verbose=False: build.LIBRARY)
    monkeypatch.setattr(build, "_run", run)
    return commands


def test_torch_calls_are_built_again_for_another_torch(compiled, monkeypatch):
    build.build_torch_calls()
    assert len(compiled) == 1
    build.build_torch_calls()
    assert len(compiled) == 1  # nothing changed
    monkeypatch.setattr(build.importlib.metadata, "version", lambda name: "99.0")
    build.build_torch_calls()
    assert len(compiled) == 2
    build.build_torch_calls()
    assert len(compiled) == 2


def test_a_torch_without_metadata_tells_its_version(monkeypatch):
    def missing(name):
        raise build.importlib.metadata.PackageNotFoundError(name)

    monkeypatch.setattr(build.importlib.metadata, "version", missing)
    assert torch.__version__ in build.torch_and_python()


def test_a_failed_build_leaves_no_claim(compiled, monkeypatch):
    build.build_torch_calls()

    def fail(command):
        raise RuntimeError("no compiler")

    monkeypatch.setattr(build, "_run", fail)
    monkeypatch.setattr(build.importlib.metadata, "version", lambda name: "99.0")
    with pytest.raises(RuntimeError, match="no compiler"):
        build.build_torch_calls()
    assert build.torch_calls_built_for() is None and os.path.exists(build.TORCH_CALLS)


def test_a_module_of_another_torch_is_not_loaded(monkeypatch):
    monkeypatch.setattr(_native, "_calls", None)
    monkeypatch.setattr(_native, "torch_calls_built_for", lambda: "torch 1.0, cpython-38")
    with pytest.raises(_native.NativeLibraryError, match="was built for torch 1.0"):
        _native.load_torch_calls()


@pytest.mark.parametrize("which", ["absent", "without headers"])
def test_without_torch_the_rest_is_built(compiled, monkeypatch, tmp_path, capsys, which):
    built = []
    monkeypatch.setattr(build, "build_library", lambda verbose=False: built.append("library"))
    monkeypatch.setattr(build, "build_harness", lambda verbose=False: built.append("harness"))
    spec = None if which == "absent" else SimpleNamespace(origin=str(tmp_path / "torch" / "__init__.py"))
    find_spec = build.importlib.util.find_spec
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: spec if name == "torch" else find_spec(name))
    build.build_all()
    assert built == ["library", "harness"] and not compiled
    assert "not built" in capsys.readouterr().err
    with pytest.raises(RuntimeError, match="no torch"):
        build.build_torch_calls()


def test_a_missing_module_fails_at_the_first_call(tmp_path):
    """In a process of its own: the package, its expert-layer modules included,
    can be imported (and documented, and tested) without the built module."""
    program = f"""
import pathlib, sys
sys.path.insert(0, {str(build.PACKAGE_DIR.parent)!r})
from kernel_mcts_b200 import _native
_native.TORCH_CALLS = pathlib.Path({str(tmp_path / "missing.so")!r})
from kernel_mcts_b200 import grouped, mxfp4
import torch
assert not hasattr(_native.torch_calls, "__wrapped__")  # looking at it loads nothing
x = torch.zeros(2, 32, dtype=torch.bfloat16)
for call in (lambda: grouped.grouped_linear(x, x, x), lambda: mxfp4.mxfp4_quantize(x)):
    try:
        call()
    except _native.NativeLibraryError as error:
        assert "not built" in str(error)
    else:
        raise SystemExit("the call did not fail")
"""
    done = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
