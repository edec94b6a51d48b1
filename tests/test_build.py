"""The build: the library does not depend on the Python binding's compiler and
headers, and the binding follows the torch and the interpreter it is built for."""

import importlib.metadata
import importlib.util
import os
import subprocess

import pytest

from conftest import PKG


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """build.py on an empty output tree, with the compilers' calls recorded."""
    spec = importlib.util.spec_from_file_location("srswa_build", os.path.join(PKG, "csrc", "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    monkeypatch.setattr(b, "BUILD", str(tmp_path / "_build"))
    monkeypatch.setattr(b, "OUT", str(tmp_path / "libsrswa.so"))
    monkeypatch.setattr(b, "BIND", str(tmp_path / "_bind.so"))
    monkeypatch.delenv("CXX", raising=False)
    b.calls, b.fail = [], ()

    def run(cmd, **kw):
        out = cmd[cmd.index("-o") + 1]
        b.calls.append(os.path.basename(out).removesuffix(".tmp"))
        if b.calls[-1] in b.fail:
            return subprocess.CompletedProcess(cmd, 1, "", "no")
        with open(out, "w") as f:
            f.write("x")
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(b.subprocess, "run", run)
    return b


def test_builds_once(tree):
    assert tree.build() == tree.OUT and os.path.exists(tree.OUT) and os.path.exists(tree.BIND)
    assert sorted(tree.calls) == sorted([s[:-3] + ".o" for s in tree.SOURCES] + ["libsrswa.so", "_bind.so"])
    tree.calls.clear()
    tree.build()
    assert tree.calls == []


def test_library_without_a_compiler_for_the_binding(tree, monkeypatch, capsys):
    monkeypatch.setenv("CXX", "/nonexistent/g++")
    assert tree.build() == tree.OUT and os.path.exists(tree.OUT)
    assert not os.path.exists(tree.BIND) and "_bind.so" in capsys.readouterr().err


def test_library_without_torch(tree, monkeypatch, capsys):
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    assert tree.build() == tree.OUT and os.path.exists(tree.OUT)
    assert not os.path.exists(tree.BIND) and "torch" in capsys.readouterr().err


def test_library_is_linked_before_a_failing_binding_raises(tree):
    tree.fail = ("_bind.so",)
    with pytest.raises(RuntimeError, match="bind.cpp"):
        tree.build()
    assert os.path.exists(tree.OUT) and not os.path.exists(tree.BIND)


@pytest.mark.parametrize("what", ["torch", "interpreter"])
def test_binding_follows_torch_and_interpreter(tree, monkeypatch, what):
    tree.build()
    tree.calls.clear()
    if what == "torch":
        monkeypatch.setattr(importlib.metadata, "version", lambda name: "9.9.9")
    else:
        var = tree.sysconfig.get_config_var
        monkeypatch.setattr(tree.sysconfig, "get_config_var", lambda k: "cpython-999" if k == "SOABI" else var(k))
    tree.build()
    assert tree.calls == ["_bind.so"]
    tree.calls.clear()
    tree.build()
    assert tree.calls == []
