"""What building the kernel library needs, and when the torch binding is rebuilt."""
import os
from pathlib import Path

import pytest

from kernelcodegen_b200 import build


def test_the_kernel_library_builds_without_torch(native_lib, monkeypatch):
    """nvcc (and g++ for the C++ operator API) is enough: the C-ABI's users need neither torch nor its binding."""
    def never(*a, **k):
        raise AssertionError("the torch binding was built")

    monkeypatch.setattr(build, "build_binding", never)
    assert build.build() == build.LIB_PATH
    assert build.build_host() == build.HOST_LIB_PATH


@pytest.fixture
def binding(tmp_path, monkeypatch):
    """A binding that is newer than its sources, and the compiler calls that build_binding makes."""
    calls = []

    def compiler(cmd, **kw):
        calls.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_text(" ".join(cmd))
        return type("Result", (), {"returncode": 0, "stdout": ""})()

    monkeypatch.setattr(build, "BINDING_PATH", tmp_path / "_torch_binding.so")
    monkeypatch.setattr(build, "shared_libstdcxx", lambda cxx: [])
    monkeypatch.setattr(build.subprocess, "run", compiler)
    build.build_binding()
    assert len(calls) == 1
    return calls


def test_a_fresh_binding_is_left_alone(binding):
    build.build_binding()
    assert len(binding) == 1


def test_the_binding_is_rebuilt_for_another_torch(binding, monkeypatch):
    import torch

    monkeypatch.setattr(torch, "__version__", "0.0.1+other")
    build.build_binding()
    assert len(binding) == 2
    build.build_binding()
    assert len(binding) == 2


def test_the_binding_is_rebuilt_for_another_python(binding, monkeypatch):
    monkeypatch.setattr(build.sys, "version", "9.9.9 (other)")
    build.build_binding()
    assert len(binding) == 2


def test_the_binding_is_rebuilt_when_its_source_is_newer(binding):
    t = (build.CSRC / "torch_binding.cpp").stat().st_mtime
    os.utime(build.BINDING_PATH, (t - 10, t - 10))
    build.build_binding()
    assert len(binding) == 2


def test_the_binding_names_what_it_was_built_with(native_lib):
    import torch

    from kernelcodegen_b200 import _torch_binding

    assert torch.__version__ in _torch_binding.built_with
