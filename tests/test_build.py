"""What the build makes anew: on copies of the build's folders, with the compilers stood in for."""

from __future__ import annotations

import importlib.metadata
import pathlib
import shutil
import subprocess
import sys
import types

import pytest

from zippel_b200 import build


@pytest.fixture()
def made(tmp_path, monkeypatch):
    """A finished build in another folder; the names of what commands make from now on."""
    build.build_library()
    shutil.copytree(build.OBJ, tmp_path / "_obj", copy_function=shutil.copy2)
    for name in ("LIB", "ROWWISE"):
        there = getattr(build, name)
        shutil.copy2(there, tmp_path / there.name)
        monkeypatch.setattr(build, name, tmp_path / there.name)
    monkeypatch.setattr(build, "OBJ", tmp_path / "_obj")
    out = []

    def run(cmd, **_):
        target = pathlib.Path(cmd[cmd.index("-o") + 1])
        target.write_bytes(b"")
        out.append(target.name)
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(subprocess, "run", run)
    return out


def test_a_finished_build_is_left_as_it_is(made):
    build.build_library()
    assert made == []


def test_the_library_is_built_without_torch(made, monkeypatch):
    """The C interface alone: the extension on torch tensors is left out, and said to be."""
    monkeypatch.setitem(sys.modules, "torch", None)        # (an import of it fails)
    for there in (build.LIB, build.ROWWISE, build.OBJ / "zp_rowwise_torch.o"):
        there.unlink()
    assert build.build_library() == build.LIB
    assert made == [build.LIB.name] and not build.ROWWISE.exists()


def test_a_call_without_the_extension_says_what_to_do(monkeypatch):
    import zippel_b200
    from zippel_b200.blocks import rowwise
    build.build_library()
    monkeypatch.setattr(rowwise, "_module", None)
    monkeypatch.delattr(zippel_b200, "_rowwise", raising=False)
    monkeypatch.setitem(sys.modules, "zippel_b200._rowwise", None)
    with pytest.raises(RuntimeError, match="zippel_b200.build"):
        rowwise.layer_norm(None)


@pytest.mark.parametrize("what", ["torch", "python"])
def test_an_extension_of_another_torch_or_python_is_built_anew(made, monkeypatch, what):
    if what == "torch":
        monkeypatch.setattr(importlib.metadata, "version", lambda name: "0.1.2")
    else:
        monkeypatch.setattr(sys, "version", sys.version + " (another build)")
    build.build_library()
    assert made == ["zp_rowwise_torch.o", build.ROWWISE.name]
    made.clear()
    build.build_library()
    assert made == []
