"""CPU: the C library is built without torch; the host binding follows the torch that is installed."""

from __future__ import annotations

import importlib.metadata
import importlib.util
import subprocess
import sys

import pytest

from conftest import ROOT


@pytest.fixture
def build(monkeypatch, tmp_path):
    """build.py with nothing to compile, and the binding's place in a folder of its own."""
    spec = importlib.util.spec_from_file_location("fa4d_build", ROOT / "fa2-with-4d-mask_b200" / "build.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(module, "SOURCES", [])
    monkeypatch.setattr(module, "BUILD", tmp_path)
    monkeypatch.setattr(module, "LIB", tmp_path / "libfa4d.so")
    monkeypatch.setattr(module, "HOST_LIB", tmp_path / "_fa4d_host.so")
    module.LIB.touch()
    return module


def test_without_torch_the_library_is_all_there_is(build, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)  # as if it were not installed
    assert build.build() == build.LIB
    assert not build.HOST_LIB.exists()
    assert "torch" in capsys.readouterr().err


def test_the_binding_is_built_again_for_another_torch(build, monkeypatch):
    compiled = []

    def run(cmd, **kw):
        compiled.append(cmd)
        build.HOST_LIB.with_suffix(".so.tmp").touch()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    build.build()
    assert len(compiled) == 1 and build.HOST_LIB.exists()
    build.build()
    assert len(compiled) == 1
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "99.0")
    build.build()
    assert len(compiled) == 2
    build.build()
    assert len(compiled) == 2
