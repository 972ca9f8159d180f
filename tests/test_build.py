"""What a build compiles: the library always, the torch module where a CUDA torch is, and neither when nothing changed.
The compilers are fakes that write their output file."""
import importlib.machinery
import importlib.util
import os
import subprocess
from pathlib import Path

import pytest

import atomflow_b200.build as B


class Tree:
    """A package folder of its own, with the commands that a build ran in it."""

    def __init__(self, tmp, monkeypatch):
        self.tmp, self.ran, self.fail, self.clock = tmp, [], (), 1_000_000_000
        pkg = tmp / "atomflow_b200"
        (pkg / "csrc").mkdir(parents=True)
        (tmp / "include").mkdir()
        for name in ("csrc/a.cu", "csrc/b.cu", "csrc/a.h", "csrc/c.cuh", "csrc/af_generate.cpp", "csrc/af_torch.cpp",
                     "../include/atomflow_b200.h"):
            self.touch(pkg / name)
        for name, value in dict(PKG=pkg, ROOT=tmp, CSRC=pkg / "csrc", LIB=pkg / "libatomflow_b200.so",
                                CLI=pkg / "af_generate", EXT=pkg / "_torch_ops.so").items():
            monkeypatch.setattr(B, name, value)
        monkeypatch.setattr(subprocess, "run", self.run)

    def touch(self, path):
        self.clock += 10
        path.write_text("")
        os.utime(path, (self.clock, self.clock))

    def run(self, cmd, check=False, cwd=None, **kw):
        out = Path(cmd[cmd.index("-o") + 1])
        self.ran.append(out.name.removesuffix(".tmp"))
        if out.name.removesuffix(".tmp") in self.fail:
            raise subprocess.CalledProcessError(1, cmd)
        self.touch(out)

    def build(self, **kw):
        """The names of what the build made."""
        self.ran = []
        B.build(**kw)
        return self.ran


LIBRARY = ["a.o", "b.o", "libatomflow_b200.so", "af_generate"]


@pytest.fixture
def tree(tmp_path, monkeypatch):
    return Tree(tmp_path, monkeypatch)


def without_torch(monkeypatch):
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None)


def test_with_torch(tree):
    pytest.importorskip("torch")
    assert tree.build() == LIBRARY + ["_torch_ops.so"]
    assert tree.build() == []
    tree.touch(B.CSRC / "c.cuh")
    assert tree.build()[:4] == LIBRARY and tree.build() == []
    assert tree.build(force=True) == LIBRARY + ["_torch_ops.so"]


def test_without_torch_a_second_build_makes_nothing(tree, monkeypatch):
    without_torch(monkeypatch)
    assert tree.build() == LIBRARY
    assert tree.build() == []
    tree.touch(B.CSRC / "a.cu")
    assert tree.build() == LIBRARY and tree.build() == []


def test_torch_installed_later(tree, monkeypatch):
    pytest.importorskip("torch")
    with monkeypatch.context() as m:
        without_torch(m)
        assert tree.build() == LIBRARY
    assert tree.build()[-1] == "_torch_ops.so" and tree.build() == []


def torch_at(monkeypatch, root, cuda):
    """A torch under `root`, built for CUDA or not."""
    (root / "lib").mkdir(parents=True, exist_ok=True)
    for name, there in (("libc10.so", True), ("libc10_cuda.so", cuda)):
        if there:
            (root / "lib" / name).write_text("")
    (root / "__init__.py").write_text("")
    spec = importlib.machinery.ModuleSpec("torch", None, origin=str(root / "__init__.py"))
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: spec)


def test_a_torch_without_cuda_is_no_torch(tree, monkeypatch):
    torch_at(monkeypatch, tree.tmp / "cpu_torch", cuda=False)
    tree.fail = ("_torch_ops.so",)                   # there is no -lc10_cuda
    assert tree.build() == LIBRARY
    assert tree.build() == []
    torch_at(monkeypatch, tree.tmp / "cuda_torch", cuda=True)
    tree.fail = ()
    assert tree.build()[-1] == "_torch_ops.so"


def test_the_module_is_rebuilt_for_another_torch_or_python(tree, monkeypatch):
    pytest.importorskip("torch")
    tree.build()
    monkeypatch.setattr(B, "torch_version", lambda: "99.0", raising=False)
    assert tree.build() == ["_torch_ops.so"] and tree.build() == []


def test_a_module_that_failed_to_compile_is_not_fresh(tree):
    """The library is replaced before the module is compiled: the old module beside the new library is stale."""
    pytest.importorskip("torch")
    tree.build()
    tree.touch(B.ROOT / "include" / "atomflow_b200.h")
    tree.fail = ("_torch_ops.so",)
    with pytest.raises(subprocess.CalledProcessError):
        tree.build()
    tree.fail = ()
    assert tree.build() == ["_torch_ops.so"] and tree.build() == []


def test_a_program_that_failed_to_link_is_not_fresh(tree):
    tree.build()
    tree.touch(B.CSRC / "a.h")
    tree.fail = ("af_generate",)
    with pytest.raises(subprocess.CalledProcessError):
        tree.build()
    tree.fail = ()
    assert "af_generate" in tree.build() and tree.build() == []


def test_only_the_module_depends_on_its_source(tree):
    pytest.importorskip("torch")
    tree.build()
    tree.touch(B.CSRC / "af_torch.cpp")
    assert tree.build() == ["_torch_ops.so"] and tree.build() == []
