"""The extension that reads tensors' descriptors is optional: where it does not
compile the library is built without it, and one of another torch is not used."""

from __future__ import annotations

import importlib.util
import sysconfig
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

CSRC = Path(__file__).resolve().parents[1] / "nanovllm-dsa-offload_amd" / "csrc"


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("nvdsa_build_for_pack", CSRC / "build.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(module, "TENSOR_PACK", tmp_path / module.TENSOR_PACK.name)
    return module


@pytest.mark.parametrize("compiler", ["false", "/nowhere/c++"])
def test_a_build_without_a_compiler_goes_on(build, compiler, tmp_path, monkeypatch, capsys):
    monkeypatch.setenv("CXX", compiler)
    old = [tmp_path / "_tensor_pack.so", build.TENSOR_PACK]
    for path in old:
        path.write_bytes(b"of before")
    build._build_tensor_pack()
    assert not any(path.exists() for path in old)   # (none of another version is left to be loaded)
    assert "warning" in capsys.readouterr().err


def test_it_carries_the_versions(build):
    from nanovllm_amd import _lib, _tensor_pack

    assert build.TENSOR_PACK.name == "_tensor_pack" + sysconfig.get_config_var("EXT_SUFFIX") == Path(_tensor_pack.__file__).name
    assert _tensor_pack.torch_version == torch.__version__
    assert _lib._native_pack is _tensor_pack.pack


def test_one_of_another_torch_is_not_used():
    from nanovllm_amd import _lib

    assert _lib._native_of(SimpleNamespace(pack=len, torch_version="1.0")) is None
    assert _lib._native_of(SimpleNamespace(pack=len)) is None
    assert _lib._native_of(SimpleNamespace(pack=len, torch_version=torch.__version__)) is len
