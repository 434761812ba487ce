"""CPU: what makes the two libraries stale, and that the C ABI library needs nothing of torch's."""

from __future__ import annotations

import ctypes
import os
import sys

import pytest
import torch

from vllm_qdq_plugin import _build, _native


def test_built_libraries_are_fresh():
    _native.lib()
    assert not _build.is_stale()
    assert _build.build_ops() == _build.TORCH_OPS_PATH and not _build.ops_are_stale()


@pytest.mark.parametrize("name,value", [("__version__", "9.9.9"), ("version.cuda", "99.9"), ("_C._GLIBCXX_USE_CXX11_ABI", False)])
def test_another_torch_makes_the_operators_stale(monkeypatch, name, value):
    _build.build_ops()
    monkeypatch.setattr(f"torch.{name}", value)
    assert _build.ops_are_stale() and not _build.is_stale()


@pytest.fixture
def small_build(monkeypatch, tmp_path):
    """Builds of one source into a folder of their own."""
    monkeypatch.setattr(_build, "LIB_DIR", tmp_path)
    monkeypatch.setattr(_build, "LIB_PATH", tmp_path / "libqdq_b200.so")
    monkeypatch.setattr(_build, "TORCH_OPS_PATH", tmp_path / "libqdq_b200_torch.so")
    monkeypatch.setattr(_build, "sources", lambda: [_build.CSRC_DIR / "abi.cu"])
    return tmp_path


@pytest.mark.parametrize("missing", ["torch", "compiler"])
def test_the_c_abi_builds_without_the_operators(monkeypatch, small_build, missing):
    if missing == "torch":
        monkeypatch.setitem(sys.modules, "torch.utils.cpp_extension", None)
        monkeypatch.delattr(torch.utils, "cpp_extension", raising=False)
    else:
        monkeypatch.setenv("CXX", "/bin/false")
    path = _build.build_native()
    assert path.exists() and ctypes.CDLL(str(path)).qdq_abi_version() > 0
    assert not _build.TORCH_OPS_PATH.exists() and not _build.is_stale()
    built = path.stat().st_mtime_ns
    assert _build.build_native() == path and path.stat().st_mtime_ns == built  # not built again for the other's sake
    with pytest.raises((RuntimeError, ImportError)):
        _build.build_ops()
    assert not list(small_build.glob(".obj.*"))


def test_a_changed_operator_source_leaves_the_c_abi_alone(monkeypatch, tmp_path):
    _build.build_ops()
    source = tmp_path / "torch_ops.cpp"
    source.write_text(_build.TORCH_OPS_SOURCE.read_text())
    os.utime(source, (2e9, 2e9))
    monkeypatch.setattr(_build, "TORCH_OPS_SOURCE", source)
    assert _build.ops_are_stale() and not _build.is_stale()


def test_compilers_without_nostdlibxx_link_without_it(monkeypatch, tmp_path):
    monkeypatch.setattr(_build, "_has_nostdlibxx", lambda cxx: False)
    _, link = _build._torch_ops_commands(tmp_path / "a.o", tmp_path / "a.so")
    assert "-nostdlib++" not in link and "-l:libstdc++.so.6" in link
    monkeypatch.undo()
    assert not _build._has_nostdlibxx("/bin/false")
