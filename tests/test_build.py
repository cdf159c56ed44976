"""The package's build: the CUDA library needs nvcc alone; the PyTorch binding is built beside
it where PyTorch and a C++ compiler are there, again for another PyTorch, and never left behind
from an older library.  Compilers are stand-ins that write what they were called for."""

import os
import stat

import pytest

from llm_training_b200 import build as b

COMPILER = """#!/bin/sh
echo "$@" >> {log}
while [ $# -gt 0 ]; do
  if [ "$1" = "-o" ]; then echo built > "$2"; fi
  shift
done
exit {rc}
"""


class Tree:
    def __init__(self, root, monkeypatch):
        self.root, self.monkeypatch = root, monkeypatch
        for d in ("csrc", "include"):
            (root / d).mkdir()
        (root / "csrc" / "a.cu").write_text("")
        (root / "csrc" / "torch_binding.cpp").write_text("")
        (root / "include" / "sqrtblock.h").write_text("")
        monkeypatch.setattr(b, "CSRC", str(root / "csrc"))
        monkeypatch.setattr(b, "INCLUDE", str(root / "include"))
        monkeypatch.setattr(b, "BUILD", str(root / "_build"))
        monkeypatch.setattr(b, "LIBDIR", str(root / "lib"))
        monkeypatch.setattr(b, "LIBPATH", str(root / "lib" / "libsqrtblock.so"))
        monkeypatch.setattr(b, "BINDINGPATH", str(root / "lib" / "sqb_torch.so"))
        monkeypatch.setenv("NVCC", self.compiler("nvcc"))
        monkeypatch.setenv("CXX", self.compiler("g++"))
        self.torch("2.11.0")

    def compiler(self, name, rc=0):
        path = self.root / name
        path.write_text(COMPILER.format(log=self.root / (name + ".log"), rc=rc))
        path.chmod(path.stat().st_mode | stat.S_IEXEC)
        return str(path)

    def torch(self, version):
        """A PyTorch of this version, or none."""
        self.monkeypatch.setattr(b, "_torch", lambda: None if version is None else (
            str(self.root / "torch"), version))

    def calls(self, name):
        log = self.root / (name + ".log")
        return log.read_text().count("\n") if log.exists() else 0

    def has(self, name):
        return (self.root / "lib" / name).exists()


@pytest.fixture
def tree(tmp_path, monkeypatch):
    return Tree(tmp_path, monkeypatch)


def test_library_and_binding(tree):
    assert b.build() == b.LIBPATH
    assert tree.has("libsqrtblock.so") and tree.has("sqb_torch.so")
    counts = tree.calls("nvcc"), tree.calls("g++")
    assert counts == (2, 1)  # one source, one link; the binding
    b.build()
    assert (tree.calls("nvcc"), tree.calls("g++")) == counts  # nothing is stale


def test_without_pytorch(tree):
    tree.torch(None)
    with pytest.warns(RuntimeWarning, match="PyTorch"):
        b.build()
    assert tree.has("libsqrtblock.so") and not tree.has("sqb_torch.so")
    assert tree.calls("g++") == 0


def test_without_a_compiler_for_the_binding(tree):
    b.build()
    tree.monkeypatch.setenv("CXX", str(tree.root / "no such compiler"))
    with pytest.warns(RuntimeWarning, match="no such compiler"):
        b.build(force=True)
    # the library is new, and the binding of the old one does not stay beside it
    assert tree.calls("nvcc") == 4
    assert tree.has("libsqrtblock.so") and not tree.has("sqb_torch.so")


def test_a_binding_that_does_not_compile(tree):
    tree.compiler("g++", rc=1)
    with pytest.raises(RuntimeError, match="failed"):
        b.build()
    assert tree.has("libsqrtblock.so") and not tree.has("sqb_torch.so")


def test_a_source_that_does_not_compile(tree):
    tree.compiler("nvcc", rc=1)
    with pytest.raises(RuntimeError, match="failed"):
        b.build()
    assert not tree.has("libsqrtblock.so")


def test_another_pytorch(tree):
    b.build()
    tree.torch("2.12.0")
    b.build()
    assert tree.calls("g++") == 2 and tree.calls("nvcc") == 2
    b.build()
    assert tree.calls("g++") == 2
    # a compile that failed is tried again
    tree.torch("2.13.0")
    tree.compiler("g++", rc=1)
    with pytest.raises(RuntimeError):
        b.build()
    tree.compiler("g++")
    b.build()
    assert tree.has("sqb_torch.so") and tree.calls("g++") == 4


def test_the_installed_pytorch_is_found():
    import torch

    where, version = b._torch()
    assert os.path.samefile(where, os.path.dirname(torch.__file__))
    assert version == torch.__version__
