"""Building the library and the paged cache's Python binding: what depends on what (runs without a GPU;
the compilers are replaced)."""

from __future__ import annotations

import importlib.metadata
import importlib.util
import subprocess
import sys
import types

import pytest

from ttspipe_b200 import build, pagedkv


@pytest.fixture()
def compilers(monkeypatch, tmp_path):
    """Every command is noted and writes what it is told to; `fails` names a program that does not."""
    ran = types.SimpleNamespace(commands=[], fails=None)

    def run(cmd, **kw):
        ran.commands.append(cmd)
        if ran.fails and ran.fails in cmd[0]:
            return subprocess.CompletedProcess(cmd, 1, "", "no")
        out = cmd[cmd.index("-o") + 1]
        open(out, "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    for name, file in (("LIB", "lib.so"), ("BIND", "bind.so")):
        monkeypatch.setattr(build, name, tmp_path / file)
    monkeypatch.setattr(build, "BUILD", tmp_path / "build")
    monkeypatch.setattr(build, "nvcc", lambda: "nvcc")
    monkeypatch.setenv("CXX", "the-cxx")
    ran.bindings = lambda: [c for c in ran.commands if c[0] == "the-cxx"]
    return ran


def test_the_library_is_built_whatever_becomes_of_the_binding(compilers):
    compilers.fails = "the-cxx"
    with pytest.raises(RuntimeError, match="the-cxx failed on pagedkv_bind.cpp"):
        build.build()
    assert build.LIB.exists() and not build.BIND.exists()


def test_without_pytorch_the_library_is_built_alone(compilers, monkeypatch, capsys):
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build() == build.LIB and build.LIB.exists()
    assert not compilers.bindings() and "PyTorch" in capsys.readouterr().err


def test_the_binding_is_built_again_for_another_pytorch_or_compiler(compilers, monkeypatch):
    build.build()
    build.build()
    assert len(compilers.bindings()) == 1
    version = importlib.metadata.version
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "9.9" if name == "torch" else version(name))
    build.build()
    build.build()
    assert len(compilers.bindings()) == 2
    monkeypatch.setenv("CXX", "/opt/the-cxx")
    build.build()
    assert compilers.commands[-1][0] == "/opt/the-cxx" and len(compilers.commands) == 3 + len(build.sources()) + 1


@pytest.mark.parametrize("error,message", [
    (ModuleNotFoundError("No module named 'ttspipe_b200._pagedkv'", name="ttspipe_b200._pagedkv"), "is not built"),
    (ImportError("cannot import name '_pagedkv' from 'ttspipe_b200'", name="ttspipe_b200"), "is not built"),
    (ImportError("_pagedkv.so: undefined symbol: _ZN3c10"), "undefined symbol: _ZN3c10"),
])
def test_a_binding_that_does_not_load_says_why(monkeypatch, tmp_path, error, message):
    import builtins

    real = builtins.__import__

    def load(name, globals=None, locals=None, fromlist=(), level=0):
        if fromlist and "_pagedkv" in fromlist:
            raise error
        return real(name, globals, locals, fromlist, level)

    monkeypatch.setattr(builtins, "__import__", load)
    monkeypatch.setattr(pagedkv, "_native", None)
    bind = tmp_path / "_pagedkv.so"
    if "undefined" in message:
        bind.touch()
    monkeypatch.setattr(build, "BIND", bind)
    with pytest.raises(RuntimeError, match=message):
        pagedkv._bound()


def test_what_is_built_needs_no_compiler(compilers, monkeypatch):
    build.build()
    ran = len(compilers.commands)
    monkeypatch.delenv("CXX")
    monkeypatch.setattr(build.shutil, "which", lambda name: None)
    assert build.build() == build.LIB and len(compilers.commands) == ran
    with pytest.raises(FileNotFoundError, match="no C"):
        build.build_binding(force=True)
