"""``b200_torch_calls.so`` is compiled against one torch: for another it is built anew, and until then it is not loaded."""

import subprocess
from types import SimpleNamespace

import pytest
import torch

import build_native
from cuda_runtime import native


@pytest.fixture
def compiler(monkeypatch):
    """Commands that would have been run; each writes what a compiler would."""
    build_native.build_torch_calls()
    ran = []

    def run(cmd, **kw):
        ran.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "wb") as f:
            f.write(b"\x7fELF" + native.torch_calls_built_for().encode() + b"\0")
        return SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(subprocess, "run", run)
    return ran


def test_the_module_is_built_again_for_another_torch(compiler, monkeypatch, tmp_path):
    copy = tmp_path / "b200_torch_calls.so"
    copy.write_bytes(build_native.CALLS_PATH.read_bytes())
    monkeypatch.setattr(build_native, "CALLS_PATH", copy)
    build_native.build_torch_calls()
    assert compiler == []
    monkeypatch.setattr(torch, "__version__", "2.99.0+cu130")
    build_native.build_torch_calls()
    assert len(compiler) == 1
    build_native.build_torch_calls()
    assert len(compiler) == 1


def test_a_module_for_another_torch_is_not_loaded(monkeypatch):
    build_native.build_torch_calls()
    monkeypatch.setattr(native, "_calls", None)
    monkeypatch.setattr(torch, "__version__", "2.99.0+cu130")
    with pytest.raises(RuntimeError, match="another torch"):
        native.torch_calls()
    monkeypatch.undo()
    assert native.torch_calls().sample_rows


@pytest.mark.parametrize("trouble", [RuntimeError("g++ failed for torch_calls.cpp"), ImportError("No module named 'torch'"), FileNotFoundError("g++")])
def test_the_library_is_built_where_the_module_cannot_be(monkeypatch, trouble):
    """The C ABI needs neither torch nor a host compiler for its headers; the calls with torch tensors say that their module is missing."""
    build_native.build()   # (nothing is compiled below)

    def fail(*a, **kw):
        raise trouble

    monkeypatch.setattr(build_native, "build_torch_calls", fail)
    with pytest.warns(UserWarning, match="b200_torch_calls.so"):
        assert build_native.build() == build_native.LIB_PATH


def test_nobody_finds_half_a_module(compiler, monkeypatch, tmp_path):
    """While it is compiled there is none, and a failed build leaves none behind."""
    target = tmp_path / "b200_torch_calls.so"
    target.write_bytes(b"of another torch")
    monkeypatch.setattr(build_native, "CALLS_PATH", target)
    write, codes = subprocess.run, [1, 0]

    def run(cmd, **kw):
        assert not target.exists()
        done = write(cmd, **kw)
        assert not target.exists()
        done.returncode = codes.pop(0)
        return done

    monkeypatch.setattr(subprocess, "run", run)
    with pytest.raises(RuntimeError, match="failed for torch_calls.cpp"):
        build_native.build_torch_calls()
    assert list(tmp_path.iterdir()) == []
    assert build_native.build_torch_calls() == target
    assert list(tmp_path.iterdir()) == [target]
