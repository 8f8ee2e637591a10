"""Where torch, Python's headers or g++ are missing the C library is built all the same, and the serving
operators say what they miss (no GPU needed)."""

import importlib.util
import os
import shutil
import sys
import sysconfig

import pytest
import torch

import llm_kernels
from conftest import PKG
from llm_kernels import _lib


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("lk_build", os.path.join(PKG, "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(module, "BINDING", str(tmp_path / "_binding.so"))
    return module


@pytest.mark.parametrize("missing", ["torch", "headers", "compiler"])
def test_build_without_what_the_extension_needs(build, missing, tmp_path, monkeypatch, capsys):
    if missing == "torch":
        find = importlib.util.find_spec
        monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    elif missing == "headers":
        monkeypatch.setattr(sysconfig, "get_paths", lambda *a: {"include": str(tmp_path)})
    else:
        monkeypatch.setattr(shutil, "which", lambda name, *a: None)
    build._build_binding(True)
    assert not os.path.exists(build.BINDING) and "_binding.so" in capsys.readouterr().err


def test_build_with_it(build):
    if build._binding_includes() is None:
        pytest.skip("no g++, Python.h or torch headers")
    build._build_binding(False)
    assert os.path.exists(build.BINDING)


def test_a_missing_extension_is_named(monkeypatch):
    monkeypatch.setattr(_lib, "_binding", None)
    monkeypatch.delattr(llm_kernels, "_binding", raising=False)
    monkeypatch.setitem(sys.modules, "llm_kernels._binding", None)
    one, cache = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 16, 2, 64, dtype=torch.float16)
    with pytest.raises(ImportError, match="build.py"):
        llm_kernels.paged_attention(torch.zeros(1, 2, 64, dtype=torch.float16), cache, cache, one[None], one)


def test_a_torch_without_exchange_functions_is_refused():
    class Old:
        pass

    with pytest.raises(ImportError, match="DLPack"):
        _lib.binding().setup(Old, *[None] * 6)
