"""Building the torch bindings: left out without torch, again for another one."""
import os
import sys
from types import SimpleNamespace

import pytest

from tokenvector.inference_b200 import build as B


@pytest.fixture
def compiler(tmp_path, monkeypatch):
    """Output folders of the test's own, and a compiler that writes an empty file; the calls of it."""
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(B, "TORCH_LIB", str(tmp_path / "_tvq_torch.so"))
    monkeypatch.setattr(B, "OBJDIR", str(tmp_path))
    monkeypatch.setattr(B.subprocess, "run", run)
    return calls


def test_a_host_without_torch_builds_the_library_alone(compiler, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    B._build_torch(force=True)
    assert not compiler and not os.path.exists(B.TORCH_LIB)
    assert "torch is not installed" in capsys.readouterr().err


def test_the_bindings_are_built_again_for_another_torch(compiler, monkeypatch):
    pytest.importorskip("torch")
    B._build_torch(force=False)
    B._build_torch(force=False)
    assert len(compiler) == 1
    monkeypatch.setattr(B.importlib.metadata, "version", lambda name: "0.0.1")
    B._build_torch(force=False)
    B._build_torch(force=False)
    assert len(compiler) == 2
    B._build_torch(force=True)
    assert len(compiler) == 3
