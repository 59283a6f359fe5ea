"""The build of the native library and of the torch extension beside it, on a small stand-in for the sources."""

import ctypes
import importlib.metadata
import os
import shutil
import sys

import pytest

from archbench_b200 import build as B

pytestmark = pytest.mark.skipif(not (shutil.which("nvcc") or os.path.exists("/usr/local/cuda/bin/nvcc")), reason="no nvcc")

EXTENSION = """
#include <Python.h>
static PyModuleDef def = {PyModuleDef_HEAD_INIT, "_torch_ops", 0, -1, 0};
PyMODINIT_FUNC PyInit__torch_ops() { return PyModule_Create(&def); }
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    for d in ("pkg/csrc", "include"):
        os.makedirs(tmp_path / d)
    (tmp_path / "include" / "gdn_b200.h").write_text("")
    (tmp_path / "pkg" / "csrc" / "a.cu").write_text('extern "C" int answer() { return 42; }\n')
    (tmp_path / "pkg" / "csrc" / "torch_ops.cpp").write_text(EXTENSION)
    pkg = tmp_path / "pkg"
    for name, path in (("PKG", pkg), ("CSRC", pkg / "csrc"), ("OBJ", pkg / "_build"), ("LIB", pkg / "libgdn_b200.so"),
                       ("TORCH_OPS", pkg / "_torch_ops.so"), ("INCLUDE", tmp_path / "include")):
        monkeypatch.setattr(B, name, str(path))
    monkeypatch.delenv("CXX", raising=False)
    return pkg


def test_library_is_built_without_a_host_compiler_for_the_extension(tree, monkeypatch, capsys):
    monkeypatch.setenv("CXX", "no-such-compiler")
    (tree / "_torch_ops.so").write_text("made elsewhere")
    assert ctypes.CDLL(B.build()).answer() == 42
    assert os.path.exists(B.TORCH_OPS) and "no-such-compiler" in capsys.readouterr().err
    os.utime(B.TORCH_OPS, (1, 1))  # of older sources
    B.build()
    assert not os.path.exists(B.TORCH_OPS)


def test_library_is_built_where_the_extension_fails(tree):
    (tree / "csrc" / "torch_ops.cpp").write_text("#error broken\n")
    with pytest.raises(RuntimeError, match="broken"):
        B.build()
    assert ctypes.CDLL(B.LIB).answer() == 42


def test_both_are_built(tree):
    assert B.build() == B.LIB and os.path.exists(B.TORCH_OPS)
    first = os.path.getmtime(B.TORCH_OPS)
    B.build()
    assert os.path.getmtime(B.TORCH_OPS) == first


@pytest.mark.parametrize("what", ["torch", "python", "compiler"])
def test_extension_is_built_again_for_another_torch_python_or_compiler(tree, monkeypatch, what):
    B.build()
    first = os.stat(B.TORCH_OPS).st_mtime_ns
    if what == "torch":
        version = importlib.metadata.version
        monkeypatch.setattr(importlib.metadata, "version", lambda name: "0.0" if name == "torch" else version(name))
    elif what == "python":
        monkeypatch.setattr(sys, "version", "another")
    else:
        monkeypatch.setenv("CXX", shutil.which("g++") + " -g0")
    B.build()
    again = os.stat(B.TORCH_OPS).st_mtime_ns
    assert again > first
    B.build()
    assert os.stat(B.TORCH_OPS).st_mtime_ns == again
