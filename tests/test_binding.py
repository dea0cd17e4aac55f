"""The compiled host side of the drafted-step operators is built again when what it was built for changes, and is not used
with another Python or torch."""

import subprocess
from types import SimpleNamespace

import pytest
import torch

from tilejax_b200 import ops
from tilejax_b200.csrc import build as builder


@pytest.fixture
def compiled(monkeypatch, tmp_path):
    """The builder with its outputs in tmp_path and a compiler that only writes a file; the list of its calls."""
    calls = []

    def run(cmd, **_):
        calls.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("compiled")
        return SimpleNamespace(returncode=0, stdout="")

    monkeypatch.setattr(builder, "BINDING", tmp_path / "_binding.so")
    monkeypatch.setattr(builder, "BINDING_KEY", tmp_path / "binding.key", raising=False)
    monkeypatch.setattr(builder, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    monkeypatch.setattr(subprocess, "run", run)
    return calls


def test_it_is_built_once(compiled):
    assert builder.build_binding() == builder.BINDING and builder.BINDING.exists()
    builder.build_binding()
    assert len(compiled) == 1


def test_it_is_built_again_for_another_torch_or_python(compiled, monkeypatch):
    import sys

    builder.build_binding()
    monkeypatch.setattr(torch, "__version__", "0.0.0+other")
    builder.build_binding()
    assert len(compiled) == 2
    monkeypatch.setattr(sys, "implementation", SimpleNamespace(**{**vars(sys.implementation), "cache_tag": "other-1"}))
    builder.build_binding()
    builder.build_binding()
    assert len(compiled) == 3


def test_it_is_built_again_when_asked(compiled):
    builder.build_binding()
    builder.build_binding(force=True)
    assert len(compiled) == 2


def test_a_module_of_another_torch_is_not_used(native, monkeypatch):
    module = pytest.importorskip("tilejax_b200._binding")
    assert ops._native() is module
    monkeypatch.setattr(ops, "_binding", None)
    monkeypatch.setattr(torch, "__version__", "0.0.0+other")
    with pytest.raises(RuntimeError, match="csrc.build"):
        ops.rpa_commit(None, None, None, None, None, None)
