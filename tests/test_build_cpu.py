"""The build: the C library needs neither torch nor g++, the torch binding follows torch's version.

The compilers are fakes that write their output file.
"""

from __future__ import annotations

import importlib.util
from pathlib import Path
from types import SimpleNamespace

import pytest

from exfold_b200 import _lib

BUILD = Path(__file__).resolve().parent.parent / "exfold-moe_b200" / "build.py"


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("exfold_b200_build_under_test", BUILD)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.OBJ, mod.LIB = tmp_path / "obj", tmp_path / "lib" / "libexfold_b200.so"
    mod.TORCH_LIB = tmp_path / "lib" / "libexfold_b200_torch.so"
    mod.TORCH_BUILT = mod.TORCH_LIB.with_suffix(".txt")
    mod.commands, mod.fails = [], lambda cmd: False

    def run(cmd, **_):
        mod.commands.append(cmd)
        if cmd[0] == "ldd":
            return SimpleNamespace(returncode=0, stdout="libstdc++.so.6 => somewhere", stderr="")
        if mod.fails(cmd):
            return SimpleNamespace(returncode=1, stdout="", stderr="no")
        Path(cmd[cmd.index("-o") + 1]).write_bytes(b"x")
        return SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(mod, "subprocess", SimpleNamespace(run=run))
    monkeypatch.setattr(mod, "nvcc", lambda: "nvcc")
    monkeypatch.setattr(mod, "torch_command", lambda: ["g++", "-o", str(mod.TORCH_LIB)])
    monkeypatch.setattr(mod, "torch_built", lambda: "torch 1, Python 3")
    return mod


def bindings(build):
    n = sum(c[0] == "g++" for c in build.commands)
    build.commands.clear()
    return n


def test_library_without_torch(build, monkeypatch, capsys):
    monkeypatch.setattr(build, "torch_built", lambda: None)
    assert build.build().exists() and not build.TORCH_LIB.exists()
    assert bindings(build) == 0 and "not built" in capsys.readouterr().out


@pytest.mark.parametrize("missing", ["torch", "g++", "libtorch_cuda"])
def test_what_a_binding_needs(missing, tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("exfold_b200_build_under_test", BUILD)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    found = mod.torch_built()
    assert found is not None and found.startswith("torch ")
    if missing == "torch":
        monkeypatch.setattr(mod.importlib.util, "find_spec", lambda name: None)
    elif missing == "g++":
        monkeypatch.setattr(mod.shutil, "which", lambda name: None)
    else:
        monkeypatch.setattr(mod.importlib.util, "find_spec",
                            lambda name: SimpleNamespace(origin=str(tmp_path / "__init__.py")))
    assert mod.torch_built() is None


def test_a_binding_that_fails_leaves_the_library(build):
    build.fails = lambda cmd: cmd[0] == "g++"
    with pytest.raises(RuntimeError, match="build step failed"):
        build.build()
    assert build.LIB.exists() and not build.TORCH_LIB.exists()


def test_binding_follows_torch(build, monkeypatch):
    build.build()
    assert build.TORCH_BUILT.read_text().strip() == "torch 1, Python 3" and bindings(build) == 1
    build.build()
    assert bindings(build) == 0
    monkeypatch.setattr(build, "torch_built", lambda: "torch 2, Python 3")
    build.build()
    assert bindings(build) == 1 and build.TORCH_BUILT.read_text().strip() == "torch 2, Python 3"
    build.TORCH_BUILT.unlink()  # of an older build
    build.build()
    assert bindings(build) == 1


def test_another_torchs_binding_is_not_loaded(tmp_path, monkeypatch):
    monkeypatch.setattr(_lib, "_torch_ops", None)
    monkeypatch.setattr(_lib, "lib", lambda: None)
    monkeypatch.setattr(_lib, "DEFAULT_PATH", tmp_path / "libexfold_b200.so")
    with pytest.raises(RuntimeError, match="missing"):
        _lib.torch_ops()
    (tmp_path / "libexfold_b200_torch.so").write_bytes(b"x")
    (tmp_path / "libexfold_b200_torch.txt").write_text("torch 1, Python 2.7\n")
    with pytest.raises(RuntimeError, match="built for torch 1"):
        _lib.torch_ops()
