"""What the build leaves where a part of it cannot be made. No compiler runs: commands write the files that they are asked for."""
import importlib.util
import json
import os
import sys

import pytest

from helpers import ROOT


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("build_under_test", os.path.join(ROOT, "triton-rs_amd", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    for name in ("LIB", "HSACO", "META", "CALLS"):
        monkeypatch.setattr(mod, name, str(tmp_path / os.path.basename(getattr(mod, name))))
    monkeypatch.setattr(mod, "BUILD", str(tmp_path / "_build"))
    monkeypatch.setattr(mod, "CALLS_OBJ", str(tmp_path / "_build" / "module" / "calls.o"))
    mod.commands = []

    def run(cmd):
        mod.commands.append(cmd)
        if mod.broken and any(mod.broken in c for c in cmd):
            raise RuntimeError("command failed")
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("new")

    mod.broken = ""
    monkeypatch.setattr(mod, "_run", run)
    for path in (mod.LIB, mod.CALLS):
        with open(path, "w") as f:
            f.write("old")
    return mod


def content(path):
    with open(path) as f:
        return f.read()


def test_all_of_it(build):
    assert build.build(verbose=False) == build.LIB
    assert content(build.LIB) == content(build.HSACO) == content(build.CALLS) == "new"
    assert [k["name"] for k in json.loads(content(build.META))["kernels"]] == ["w4a16_gptq_gemm_typed", "awq_gemm_int4_typed"]


def test_without_torch(build, monkeypatch, capsys):
    """The library, the code object and its metadata need hipcc alone; the Python package's module is left out, and says so."""
    monkeypatch.setitem(sys.modules, "torch", None)   # (import torch raises ImportError)
    assert build.build() == build.LIB
    assert content(build.LIB) == content(build.HSACO) == "new" and json.loads(content(build.META))["kernels"]
    assert not os.path.exists(build.CALLS)            # an older one is of another library
    assert "_calls.so is not built: torch" in capsys.readouterr().out
    assert all(c[0] == build.HIPCC for c in build.commands)


@pytest.mark.parametrize("broken", ["calls.cpp", "-ltorch_python"])
def test_module_that_does_not_build(build, broken):
    build.broken = broken
    with pytest.raises(RuntimeError, match="command failed"):
        build.build()
    assert content(build.LIB) == content(build.HSACO) == "new" and json.loads(content(build.META))["kernels"]
    assert not os.path.exists(build.CALLS)


def test_library_that_does_not_build(build):
    build.broken = "norm.hip"
    with pytest.raises(RuntimeError, match="command failed"):
        build.build()
    assert content(build.LIB) == "old"
