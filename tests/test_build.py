"""The build: what needs torch, and what makes it stale."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_the_engine_builds_without_torch(tmp_path):
    """Where torch cannot be imported only the torch binding is left out."""
    code = f"""
import sys
sys.modules["torch"] = None
from pathlib import Path
from ggmlc_b200 import build
build.BINDING = Path({str(tmp_path / "_kv_q4.so")!r})
assert build.build() == build.LIB and build.LIB.exists()
assert build.build_torch_binding(force=True) is None and not build.BINDING.exists()
import ggmlc_b200._runtime
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_the_torch_binding_follows_torch(tmp_path, monkeypatch):
    """Built again for another torch or interpreter, not for the same."""
    pytest.importorskip("torch")
    from ggmlc_b200 import build

    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_bytes(b"built")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build, "BINDING", tmp_path / "_kv_q4.so")
    monkeypatch.setattr(build, "BINDING_FOR", tmp_path / "_kv_q4.for")
    monkeypatch.setattr(build.subprocess, "run", run)
    for against, built in (("torch A", 1), ("torch A", 1), ("torch B", 2), ("torch B", 2)):
        monkeypatch.setattr(build, "torch_build", lambda: against)
        assert build.build_torch_binding() == build.BINDING
        assert len(calls) == built
    monkeypatch.undo()
    assert build.torch_build() == build.torch_build() and "2" in build.torch_build()
