"""When build.py builds the tensor-level callers (_torch_ops.so): not at all without PyTorch
(the C ABI library is complete without them), again for another PyTorch or Python."""
import importlib.util
import subprocess
import sys
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parents[1] / "obsidian-memory-transformer_b200"


@pytest.fixture
def recipe(tmp_path, monkeypatch):
    """build.py with its outputs in tmp_path and a compiler that only writes its output."""
    spec = importlib.util.spec_from_file_location("ltm_build_under_test", PKG / "build.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.OPS, m.OPS_FOR = tmp_path / "_torch_ops.so", tmp_path / "b" / "torch_ops.for"
    m.ran = []

    def run(cmd, **kw):
        m.ran.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_text("built")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(m.subprocess, "run", run)
    return m


def test_without_pytorch(recipe, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)  # not found, import torch fails
    assert recipe.build_torch_ops() is None and not recipe.ran and not recipe.OPS.exists()
    assert "no PyTorch" in capsys.readouterr().err


def test_library_is_built_without_pytorch(recipe, monkeypatch, tmp_path):
    src = tmp_path / "csrc"
    src.mkdir()
    (src / "a.cu").write_text("")
    recipe.CSRC, recipe.BUILD, recipe.LIB = src, tmp_path / "b", tmp_path / "lib.so"
    monkeypatch.setitem(sys.modules, "torch", None)
    assert recipe.build() == recipe.LIB and recipe.LIB.exists() and len(recipe.ran) == 2


def test_built_again_when_pytorch_changes(recipe, monkeypatch):
    assert recipe.build_torch_ops() == recipe.OPS and len(recipe.ran) == 1
    recipe.build_torch_ops()
    assert len(recipe.ran) == 1
    here = recipe.torch_here()
    monkeypatch.setattr(recipe, "torch_here", lambda: ("0.0.0+other", here[1]))
    recipe.build_torch_ops()
    assert len(recipe.ran) == 2
    recipe.build_torch_ops()
    assert len(recipe.ran) == 2
    recipe.OPS_FOR.unlink()  # built by an older recipe: unknown
    recipe.build_torch_ops()
    assert len(recipe.ran) == 3
    recipe.build_torch_ops(force=True)
    assert len(recipe.ran) == 4


def test_headers_of_the_toolkit(recipe):
    assert (recipe.cuda_include() / "cuda_runtime_api.h").exists()
