"""The build recipe with its compilers faked: the library does not depend on torch, and the
torch module belongs to one Python."""

import subprocess
import sysconfig
from pathlib import Path

import pytest

from yufmusicgen_b200 import build as b


@pytest.fixture
def recipe(tmp_path, monkeypatch):
    """``build`` in an empty folder; ``ran`` collects its commands, ``fail`` names a program to fail."""
    made = {"ran": [], "fail": None}

    def run(cmd, **_):
        made["ran"].append([str(c) for c in cmd])
        bad = made["fail"] is not None and made["fail"] in Path(cmd[0]).name
        if not bad:
            Path(cmd[cmd.index("-o") + 1]).write_bytes(b"")
        return subprocess.CompletedProcess(cmd, int(bad), "", "no such header" if bad else "")

    monkeypatch.setattr(subprocess, "run", run)
    monkeypatch.setattr(b, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    monkeypatch.setattr(b, "_sources", lambda: [b.CSRC / "capi.cu"])
    monkeypatch.setattr(b, "OUT_DIR", tmp_path / "_build")
    monkeypatch.setattr(b, "LIB", tmp_path / "libyufb200.so")
    monkeypatch.setattr(b, "TORCH_MODULE", tmp_path / b.TORCH_MODULE.name)
    return made


def test_both_are_built_and_only_once(recipe):
    assert b.build() == b.LIB
    assert b.LIB.exists() and b.TORCH_MODULE.exists()
    n = len(recipe["ran"])
    b.build()
    assert len(recipe["ran"]) == n


def test_the_library_is_built_where_torch_is_not(recipe, monkeypatch, capsys):
    monkeypatch.setattr(b, "_torch_dir", lambda: None)
    assert b.build() == b.LIB and b.LIB.exists() and not b.TORCH_MODULE.exists()
    assert "torch" in capsys.readouterr().err


def test_a_failure_of_the_torch_module_comes_after_the_library(recipe):
    recipe["fail"] = "g++"
    with pytest.raises(RuntimeError, match="no such header"):
        b.build()
    assert b.LIB.exists() and not b.TORCH_MODULE.exists()


def test_the_torch_module_belongs_to_one_python(recipe, monkeypatch):
    assert b.TORCH_MODULE.name == "_yuf_torch" + sysconfig.get_config_var("EXT_SUFFIX")
    b.build()
    n = len(recipe["ran"])
    monkeypatch.setattr(b, "TORCH_MODULE", b.TORCH_MODULE.with_name("_yuf_torch.cpython-399-other.so"))
    b.build()
    assert b.TORCH_MODULE.exists()
    assert [c[0] for c in recipe["ran"][n:]] == ["g++", "g++"]  # compiled again, not only linked


def test_a_missing_torch_is_found_missing(monkeypatch):
    monkeypatch.setattr(b.importlib.util, "find_spec", lambda name: None)
    assert b._torch_dir() is None
