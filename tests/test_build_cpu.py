"""CPU: the C library is built and linked with nvcc alone; the Python binding beside it fails loudly, but not in the
library's way."""
from __future__ import annotations

import importlib.util
import subprocess
import sys

import pytest

from conftest import ROOT


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("kea_build", ROOT / "kea-kernels_b200" / "build.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.ran = []

    def fake(cmd, **_):
        module.ran.append(cmd)
        missing = any(str(a).endswith("binding.cpp") for a in cmd)
        return subprocess.CompletedProcess(cmd, 1 if missing and module.refuse else 0, "", "no headers" if missing else "")

    module.refuse = False
    monkeypatch.setattr(module.subprocess, "run", fake)
    monkeypatch.setattr(module, "nvcc", lambda: "nvcc")
    return module


def linked(module):
    return [cmd for cmd in module.ran if "-shared" in cmd and str(module.OUT) in cmd]


def test_library_and_binding(build):
    assert build.build(force=True) == build.OUT
    assert len(linked(build)) == 1 and any(str(build.BINDING) in cmd for cmd in build.ran)


def test_library_without_a_compiler_for_the_binding(build):
    build.refuse = True
    with pytest.raises(RuntimeError, match="binding"):
        build.build(force=True)
    assert len(linked(build)) == 1


def test_library_without_torch(build, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build(force=True) == build.OUT
    assert len(linked(build)) == 1 and not any(str(build.BINDING) in cmd for cmd in build.ran)
    assert "only the C library" in capsys.readouterr().err
