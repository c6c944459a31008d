"""What `python -m sirius_b200._build` compiles again, and in which order: the native front end follows the torch and the interpreter
it was built for, and the library comes about whether or not the front end does. No compiler runs here."""
import importlib.util
import subprocess
import types

import pytest

from sirius_b200 import _build


class Compilers:
    """Stands in for subprocess.run: keeps the commands and makes their outputs."""

    def __init__(self):
        self.commands, self.failing = [], None

    def __call__(self, cmd, **kw):
        out = cmd[cmd.index("-o") + 1]
        self.commands.append((cmd[0].rsplit("/", 1)[-1], out.rsplit("/", 1)[-1]))
        if self.failing is not None and out.endswith(self.failing):
            return types.SimpleNamespace(returncode=1, stdout="", stderr="no such header\n")
        open(out, "w").close()
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    def made(self, name):
        return sum(out == name for _, out in self.commands)


@pytest.fixture
def tree(tmp_path, monkeypatch):
    pkg = tmp_path / "pkg"
    src = pkg / "csrc" / "binding"
    src.mkdir(parents=True)
    (tmp_path / "include").mkdir()
    (tmp_path / "include" / "a.h").write_text("")
    (src.parent / "a.cu").write_text("")
    (src / "ops_module.cpp").write_text("")
    for name, value in (("PKG", pkg), ("CSRC", src.parent), ("BUILD", pkg / "build"), ("LIB", pkg / "libsirius_b200.so"),
                        ("BINDING_SRC", src / "ops_module.cpp"), ("BINDING", pkg / "_ops_native.so")):
        monkeypatch.setattr(_build, name, value)
    run = Compilers()
    monkeypatch.setattr(subprocess, "run", run)
    return run


def test_nothing_is_built_twice(tree):
    for _ in range(3):
        assert _build.build() == _build.LIB
    assert tree.made("_ops_native.so") == 1 and tree.made("libsirius_b200.so") == 1 and tree.made("a.o") == 1
    _build.build(force=True)
    assert tree.made("_ops_native.so") == 2


@pytest.mark.parametrize("what", ["torch", "interpreter", "flags"])
def test_another_torch_or_interpreter_builds_the_front_end_again(tree, monkeypatch, what):
    import importlib.metadata
    import sysconfig
    _build.build()
    if what == "torch":
        monkeypatch.setattr(importlib.metadata, "version", lambda name: "9.9.9+cu999")
    elif what == "interpreter":
        real = sysconfig.get_config_var
        monkeypatch.setattr(sysconfig, "get_config_var", lambda k: "cpython-399-x86_64" if k == "SOABI" else real(k))
    else:
        monkeypatch.setattr(_build, "NVCC", "/elsewhere/cuda/bin/nvcc")   # its headers are on the command line
    _build.build()
    assert tree.made("_ops_native.so") == 2 and tree.made("a.o") == 1
    _build.build()
    assert tree.made("_ops_native.so") == 2


def test_the_library_needs_no_torch(tree, monkeypatch, capsys):
    real = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else real(name, *a))
    assert _build.build() == _build.LIB and _build.LIB.exists()
    assert not _build.BINDING.exists()
    assert "torch" in capsys.readouterr().err


def test_the_library_is_linked_before_the_front_end_fails(tree):
    tree.failing = "_ops_native.so"
    with pytest.raises(RuntimeError, match="ops_module.cpp"):
        _build.build()
    assert _build.LIB.exists()
    tree.failing = None
    _build.build()
    assert _build.BINDING.exists()
    _build.build()
    assert tree.made("_ops_native.so") == 2
