"""When the host module of the attention calls is compiled again (no compiler runs: a stand-in records the commands)."""
import os
import subprocess
import sys
import sysconfig

import pytest
import torch

from mingmoe import build as B


@pytest.fixture
def runs(monkeypatch, tmp_path):
    """Commands that build_host ran, in a folder of its own."""
    out, ran = tmp_path / "_attention_host.so", []

    def run(cmd, **kw):
        ran.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").write("so")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(B, "HOST_OUT", str(out))
    monkeypatch.setattr(B, "BUILD", str(tmp_path / "_build"))
    monkeypatch.setattr(B.subprocess, "run", run)
    return ran


def test_compiled_once(runs):
    assert B.build_host() == B.HOST_OUT and os.path.exists(B.HOST_OUT)
    B.build_host()
    assert len(runs) == 1
    B.build_host(force=True)
    assert len(runs) == 2


def test_compiled_again_for_another_torch(runs, monkeypatch):
    B.build_host()
    monkeypatch.setattr(torch, "__version__", "9.9.0")
    B.build_host()
    assert len(runs) == 2


def test_compiled_again_for_another_python(runs, monkeypatch):
    B.build_host()
    paths = dict(sysconfig.get_paths(), include="/elsewhere/include/python9.9")
    monkeypatch.setattr(sysconfig, "get_paths", lambda: paths)
    B.build_host()
    assert len(runs) == 2


def test_compiled_again_where_only_the_module_is_left(runs):
    """A module of unknown origin beside no record of what it was compiled for."""
    open(B.HOST_OUT, "w").write("so")
    B.build_host()
    assert len(runs) == 1
