"""When the torch binding is built (rustane_b200/build.py), with the compiler replaced by a function that writes its output."""
import subprocess
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest

from rustane_b200 import build as b


@pytest.fixture
def fake(monkeypatch, tmp_path):
    runs = []

    def run(cmd, **kw):
        runs.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_text("built")
        return SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(b, "BUILD", tmp_path)
    monkeypatch.setattr(b, "TORCH_EXT", tmp_path / "_torch_ops.so")
    monkeypatch.setattr(subprocess, "run", run)
    return runs


def test_the_binding_is_built_again_for_another_torch(fake, monkeypatch):
    torch = pytest.importorskip("torch")
    assert b.build_torch_ext() == b.TORCH_EXT and len(fake) == 1
    assert b.build_torch_ext() == b.TORCH_EXT and len(fake) == 1
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    assert b.build_torch_ext() == b.TORCH_EXT and len(fake) == 2
    assert b.build_torch_ext() == b.TORCH_EXT and len(fake) == 2
    monkeypatch.setattr(b, "INCLUDE", b.INCLUDE.parent / "include" / ".." / "include")  # another command
    b.build_torch_ext()
    assert len(fake) == 3


def test_the_library_builds_without_torch(fake, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)  # import torch raises ImportError
    assert b.build_torch_ext() is None and not fake
    assert "torch" in capsys.readouterr().out
