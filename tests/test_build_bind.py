"""The build of the tensor binding: left out where torch cannot be imported, and rebuilt for another torch or interpreter."""
from __future__ import annotations

import json
import os
import shutil
import subprocess
import sys

import pytest

from matmulfreellmcpu_b200 import _lib
from matmulfreellmcpu_b200 import build as B
from conftest import ROOT


@pytest.fixture
def elsewhere(tmp_path, monkeypatch):
    """The binding's files in a folder of the test's, as they are built."""
    for name in ("BIND", "BIND_FOR"):
        to = str(tmp_path / os.path.basename(getattr(B, name)))
        shutil.copy2(getattr(B, name), to)
        monkeypatch.setattr(B, name, to)
    return tmp_path


def recorded(monkeypatch):
    """Compiler calls, none of which runs."""
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(B.subprocess, "run", run)
    return calls


def test_the_library_and_the_cli_build_without_torch():
    """build() in an interpreter that has no torch ends well, with a word about what it left out (whatever it would compile
    anew is not compiled here)."""
    code = ("import sys, types; sys.modules['torch'] = None\n"
            "from matmulfreellmcpu_b200 import build\n"
            "build.subprocess = types.SimpleNamespace(run=lambda *a, **k: types.SimpleNamespace(returncode=0, stdout='', stderr=''))\n"
            "assert build.build() == build.LIB and build.build_bind() is None\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert "tensor binding not built" in r.stderr


def test_a_binding_for_this_torch_is_kept(elsewhere, monkeypatch):
    calls = recorded(monkeypatch)
    os.utime(B.BIND)
    assert B.build_bind() == B.BIND and calls == []


@pytest.mark.parametrize("key,value", [("torch", "0.0"), ("python", "cpython-27"), ("cxx11_abi", 7), (None, None)])
def test_a_binding_for_another_torch_or_python_is_rebuilt_and_not_loaded(elsewhere, monkeypatch, key, value):
    calls = recorded(monkeypatch)
    os.utime(B.BIND)
    if key is None:
        os.remove(B.BIND_FOR)  # of a build that kept no record
    else:
        with open(B.BIND_FOR) as f:
            target = json.load(f)
        with open(B.BIND_FOR, "w") as f:
            json.dump({**target, key: value}, f)
    monkeypatch.setattr(_lib, "_BIND", None)
    with pytest.raises(ImportError, match="matmulfreellmcpu_b200.build"):
        _lib.bind()
    B.build_bind()
    assert len(calls) == 1 and B.bind_built_for() == B.bind_target()
