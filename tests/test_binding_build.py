"""The torch binding belongs to one torch and one Python; the library without it still builds and works."""
import sys

import pytest
import torch

import npu_offload_b200 as nob
from npu_offload_b200 import build, moe


def test_the_binding_in_the_tree_is_of_this_torch_and_python():
    path = build.binding_path()
    assert torch.__version__ in path and sys.implementation.cache_tag in path
    assert build.build_binding() == path


@pytest.mark.parametrize("what", ["torch", "python"])
def test_a_binding_of_another_version_is_not_loaded(monkeypatch, what):
    """It may differ in the layout of every object that it is handed."""
    if what == "torch":
        monkeypatch.setattr(torch, "__version__", "9.9.9")
    else:
        monkeypatch.setattr(sys.implementation, "cache_tag", "cpython-999")
    monkeypatch.setattr(moe, "_calls", None)
    p = object.__new__(nob.MoEDataPlane)
    p.H, p.F, p.E, p.K, p._h, p._index, p._plane = 256, 64, 8, 2, None, 0, None
    p.device = torch.device("cpu")
    monkeypatch.setattr(moe, "_raw_stream", lambda index: 0)
    with pytest.raises(ImportError, match="npu_offload_b200.build"):
        p.quantize_fp8(torch.zeros(4, 32))


@pytest.mark.parametrize("lacking", ["compiler", "torch", "headers"])
def test_the_library_builds_without_what_the_binding_needs(monkeypatch, lacking, capsys):
    """Only the e4m3 and balance-loss calls from Python need the binding."""
    monkeypatch.setattr(build, "build_library", lambda *a, **k: "the library")
    if lacking == "compiler":
        monkeypatch.setattr(build, "CXX", "/nowhere/g++")
    elif lacking == "torch":
        monkeypatch.setitem(sys.modules, "torch", None)
    else:
        monkeypatch.setattr(build, "CXX", "false")  # what a compiler returns that finds no headers
    assert build.build(force=True) == "the library"
    assert "binding" in capsys.readouterr().err
    with pytest.raises(Exception):
        build.build_binding(force=True)
