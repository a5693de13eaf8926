"""The build script: the C library needs nvcc alone; the Python module of the operators does not stop it,
and follows the installed torch."""
import importlib.util
import subprocess
import sys
from types import SimpleNamespace

import pytest

from conftest import ROOT


@pytest.fixture
def build(tmp_path, monkeypatch):
    """The script over an empty tree with one source; commands are recorded, and make their output files."""
    spec = importlib.util.spec_from_file_location("build_under_test", ROOT / "tekken8-agent_b200" / "build.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    for folder in ("csrc", "include", "bindings", "t8b"):
        (tmp_path / folder).mkdir()
    for name in ("csrc/one.cu", "csrc/common.cuh", "include/t8b.h", "bindings/operators.cpp"):
        (tmp_path / name).write_text("")
    monkeypatch.setattr(module, "ROOT", tmp_path)
    monkeypatch.setattr(module, "CSRC", tmp_path / "csrc")
    monkeypatch.setattr(module, "BUILD", tmp_path / "_build")
    monkeypatch.setattr(module, "LIB", tmp_path / "lib" / "libt8b.so")
    monkeypatch.setattr(module, "MODULE_SOURCE", tmp_path / "bindings" / "operators.cpp")
    monkeypatch.setattr(module, "MODULE", tmp_path / "t8b" / "_operators.so")
    ran = []

    def run(command, check):
        from pathlib import Path
        assert check
        out = Path(command[command.index("-o") + 1])
        ran.append(out.name)
        out.write_text("")
        return SimpleNamespace(returncode=0)

    monkeypatch.setattr(subprocess, "run", run)
    return SimpleNamespace(script=module, ran=ran, tmp=tmp_path, monkeypatch=monkeypatch)


def test_the_library_is_linked_without_torch(build, capsys):
    build.monkeypatch.setitem(sys.modules, "torch", None)  # importing it raises ImportError
    lib = build.script.build()
    assert lib.exists() and build.ran == ["one.o", "libt8b.so"]
    assert "_operators" in capsys.readouterr().err


def test_the_module_follows_the_library_and_is_not_rebuilt_for_nothing(build):
    build.script.build()
    assert sorted(build.ran) == ["_operators.so", "libt8b.so", "one.o"]
    build.script.build()
    assert len(build.ran) == 3


def test_another_torch_rebuilds_the_module(build):
    import importlib.metadata
    build.script.build()
    build.monkeypatch.setattr(importlib.metadata, "version", lambda name: "0.0.1+other")
    build.script.build()
    assert build.ran[3:] == ["_operators.so"]


def test_a_module_that_does_not_compile_is_an_error_and_the_library_is_there(build):
    def fails(command, check):
        if "_operators.so" in str(command):
            raise subprocess.CalledProcessError(1, command)
        return run(command, check)

    run = subprocess.run
    build.monkeypatch.setattr(subprocess, "run", fails)
    with pytest.raises(subprocess.CalledProcessError):
        build.script.build()
    assert build.ran == ["one.o", "libt8b.so"]
