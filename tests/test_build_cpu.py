"""When the extension module is compiled again (nlearn_b200/build.py)."""
import os
import subprocess

import pytest

from nlearn_b200 import build as B


@pytest.fixture
def compiler(tmp_path, monkeypatch):
    """A build tree of its own, and a compiler that writes its output and is counted."""
    runs = []

    def run(cmd, **kw):
        runs.append(cmd)
        B.EXT.write_bytes(b"module")
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(B, "EXT", tmp_path / "_ops.so")
    monkeypatch.setattr(B, "BUILD_DIR", tmp_path)
    monkeypatch.setattr(B.subprocess, "run", run)
    return runs


def test_another_torch_compiles_again(compiler, monkeypatch):
    import torch
    assert B._build_ext().startswith("compiled") and B._build_ext().startswith("up to date")
    monkeypatch.setattr(torch, "__version__", "9.9.9+other")
    assert B._build_ext().startswith("compiled") and B._build_ext().startswith("up to date")
    monkeypatch.setattr(B.sys, "version", "9.9 (other)")
    assert B._build_ext().startswith("compiled")
    assert len(compiler) == 3


def test_newer_sources_compile_again(compiler):
    B._build_ext()
    t = B.EXT_SRC.stat().st_mtime - 10
    os.utime(B.EXT, (t, t))
    assert B._build_ext().startswith("compiled") and len(compiler) == 2
