"""The native binding is built again, and not loaded, when torch is not the one it was
built against."""

import subprocess
import types

import pytest
import torch

from litevllm_b200 import _lib, build


@pytest.fixture
def compiled(monkeypatch, tmp_path):
    """Commands of build_spec, which write to a folder of the test's."""
    monkeypatch.setattr(build, "SPEC", tmp_path / "_spec.so")
    monkeypatch.setattr(build, "BUILD", tmp_path / "_build")
    ran = []

    def run(cmd, **kw):
        ran.append(cmd)
        (tmp_path / "_spec.so.tmp").write_bytes(b"built")
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(subprocess, "run", run)
    return ran


def test_binding_is_built_once(compiled):
    for _ in range(2):
        assert build.build_spec().read_bytes() == b"built"
    assert len(compiled) == 1
    build.build_spec(force=True)
    assert len(compiled) == 2


@pytest.mark.parametrize("what", ["torch", "python", "compiler", "no record"])
def test_binding_is_built_again(compiled, monkeypatch, what):
    build.build_spec()
    if what == "torch":
        monkeypatch.setattr(torch, "__version__", "9.9.9+cu999")
    elif what == "python":
        monkeypatch.setattr(build.sys, "version", "3.99")
    elif what == "compiler":
        monkeypatch.setenv("CXX", "another-g++")
    else:
        (build.BUILD / "_spec.txt").unlink()
    build.build_spec()
    build.build_spec()
    assert len(compiled) == 2


def test_binding_of_another_torch_is_refused(monkeypatch):
    assert _lib.spec_module().torch_version == torch.__version__
    monkeypatch.setattr(torch, "__version__", "9.9.9+cu999")
    with pytest.raises(_lib.LiteKernError, match="does not fit torch 9.9.9"):
        _lib.spec_module()


def test_binding_that_does_not_load_is_refused(monkeypatch, tmp_path):
    bad = tmp_path / "_spec.so"
    bad.write_bytes(b"not a library")
    monkeypatch.setattr(_lib, "SPEC_PATH", bad)
    with pytest.raises(_lib.LiteKernError, match="does not fit torch"):
        _lib.spec_module()
