"""_host.so is made again when what it was made by has changed."""
import importlib.util
import os
import sys

import pytest
import torch

from conftest import PKG


@pytest.fixture()
def build(tmp_path, monkeypatch):
    """build.py with everything in place, its commands noted instead of run."""
    spec = importlib.util.spec_from_file_location("smoe_build_under_test", os.path.join(PKG, "build.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.commands = []

    def note(command):
        m.commands.append(command)
        open(command[command.index("-o") + 1], "w").close()

    monkeypatch.setattr(m.subprocess, "check_call", note)
    monkeypatch.setattr(m, "_stale", lambda target, deps: not os.path.exists(target))
    (tmp_path / "sonicmoe").mkdir()
    (tmp_path / "build").mkdir()
    for src in m.SOURCES:
        (tmp_path / "build" / src.replace(".cu", ".o")).touch()
    monkeypatch.setattr(m, "HERE", str(tmp_path))
    monkeypatch.setattr(m, "OUT", str(tmp_path / "sonicmoe" / "libsmoe_b200.so"))
    monkeypatch.setattr(m, "HOST_OUT", str(tmp_path / "sonicmoe" / "_host.so"))
    monkeypatch.setattr(m, "HOST_MADE", str(tmp_path / "build" / "_host.command"), raising=False)
    open(m.OUT, "w").close()
    return m


def made(m):
    m.commands.clear()
    m.build()
    return [c for c in m.commands if m.HOST_OUT in c]


def test_another_pytorch_python_or_compiler(build, monkeypatch):
    assert len(made(build)) == 1 and not made(build)
    monkeypatch.setattr(torch, "__version__", "99.0+cu1")
    assert len(made(build)) == 1 and not made(build)
    monkeypatch.setattr(sys, "version", "4.0")
    assert len(made(build)) == 1 and not made(build)
    monkeypatch.setenv("CXX", "another-g++")
    assert [c[0] for c in made(build)] == ["another-g++"] and not made(build)
    os.remove(build.HOST_OUT)
    assert len(made(build)) == 1 and not made(build)


def test_a_build_that_failed_is_not_taken_for_one(build, monkeypatch):
    assert len(made(build)) == 1
    note, version = build.subprocess.check_call, torch.__version__

    def fails(command):
        raise RuntimeError("no compiler")

    monkeypatch.setattr(torch, "__version__", "99.0+cu1")
    monkeypatch.setattr(build.subprocess, "check_call", fails)
    with pytest.raises(RuntimeError):
        build.build()
    monkeypatch.setattr(torch, "__version__", version)       # (what the failed one left may be anything)
    monkeypatch.setattr(build.subprocess, "check_call", note)
    assert len(made(build)) == 1 and not made(build)


def test_without_pytorch_the_library_of_the_c_entry_points_is_built(build, monkeypatch):
    monkeypatch.setitem(sys.modules, "torch", None)
    os.remove(build.OUT)
    assert build.build() == build.OUT and os.path.exists(build.OUT) and not os.path.exists(build.HOST_OUT)
