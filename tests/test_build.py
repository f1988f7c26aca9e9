"""build.py: what the library and its PyTorch binding need."""

import importlib.util
import sys
from pathlib import Path

import pytest

SOURCE = Path(__file__).resolve().parent.parent / "jittor-flow2surf_b200" / "build.py"


@pytest.fixture
def native_build(monkeypatch, tmp_path):
    """build.py on a tree of its own: one source, compiled and linked by recorded commands."""
    spec = importlib.util.spec_from_file_location("native_build", SOURCE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    for name in ("CSRC", "INCLUDE", "BUILD"):
        (tmp_path / name).mkdir()
        monkeypatch.setattr(module, name, tmp_path / name)
    (tmp_path / "CSRC" / "one.cu").write_text("")
    monkeypatch.setattr(module, "LIBRARY", tmp_path / "library.so")
    monkeypatch.setattr(module, "BINDING", tmp_path / "binding.so")
    monkeypatch.setattr(module, "BINDING_SOURCE", tmp_path / "CSRC" / "binding.cpp")
    (tmp_path / "CSRC" / "binding.cpp").write_text("")
    commands = []

    class Done:
        returncode, stdout, stderr = 0, "", ""

    def run(cmd, **kwargs):
        commands.append(cmd[0].rsplit("/", 1)[-1])
        Path(cmd[cmd.index("-o") + 1]).write_text("")
        return Done

    monkeypatch.setattr(module.subprocess, "run", run)
    monkeypatch.setattr(module, "nvcc", lambda: "/cuda/bin/nvcc")
    return module, commands


def test_library_and_binding(native_build):
    module, commands = native_build
    assert module.binding_lacks() is None
    assert module.build() == module.LIBRARY
    assert sorted(commands) == ["g++", "g++", "nvcc", "nvcc"] and module.BINDING.exists()


@pytest.mark.parametrize("missing", ["torch", "Python.h", "g++"])
def test_library_needs_no_torch(native_build, monkeypatch, tmp_path, capsys, missing):
    module, commands = native_build
    if missing == "torch":
        monkeypatch.setitem(sys.modules, "torch", None)
        find = importlib.util.find_spec
        monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    elif missing == "Python.h":
        monkeypatch.setattr(module.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    else:
        which = module.shutil.which
        monkeypatch.setattr(module.shutil, "which", lambda name: None if name == "g++" else which(name))
    assert module.build() == module.LIBRARY
    assert commands == ["nvcc", "nvcc"] and module.LIBRARY.exists() and not module.BINDING.exists()
    assert missing in capsys.readouterr().err
