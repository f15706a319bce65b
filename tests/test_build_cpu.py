"""When the native binding is built anew, and that the library is built without it."""
import os
import subprocess

import pytest
import torch

from conftest import load_pkg


@pytest.fixture
def b(tmp_path, monkeypatch):
    """The build module with a binding of its own, up to date, and no compiler behind it."""
    mod = load_pkg("build")
    source, header = tmp_path / "x.cpp", tmp_path / "x.h"
    for p in (source, header):
        p.write_text("")
        os.utime(p, (1000, 1000))
    binding = tmp_path / "_b2torch.so"
    binding.write_bytes(b"\x7fELF..." + mod.binding_stamp().encode() + b"\0")
    monkeypatch.setattr(mod, "BINDING", binding)
    monkeypatch.setattr(mod, "BINDING_SOURCE", source)
    monkeypatch.setattr(mod, "BINDING_HEADERS", [header])
    monkeypatch.setattr(mod, "_build_library", lambda force, verbose: "library")
    return mod


def _compiler(monkeypatch, code):
    """subprocess.Popen as a compiler that exits with `code`; the commands it got."""
    seen = []

    def popen(cmd, **kw):
        seen.append(cmd)
        out = cmd[cmd.index("-o") + 1]
        if code == 0:
            open(out, "wb").write(b"new")
        return type("Proc", (), {"returncode": code, "communicate": lambda self: ("no such header", None)})()
    monkeypatch.setattr(subprocess, "Popen", popen)
    return seen


def test_binding_is_up_to_date(b, monkeypatch):
    assert b.binding_matches(b.BINDING) and not b.binding_needs_build()
    seen = _compiler(monkeypatch, 0)
    assert b.build() == "library" and not seen


@pytest.mark.parametrize("what", ["source", "header", "torch", "python", "missing"])
def test_binding_is_built_anew(b, monkeypatch, what):
    if what == "source":
        os.utime(b.BINDING_SOURCE)
        os.utime(b.BINDING, (2000, 2000))
    elif what == "header":
        os.utime(b.BINDING_HEADERS[0])
        os.utime(b.BINDING, (2000, 2000))
    elif what == "torch":
        monkeypatch.setattr(torch, "__version__", "2.12.0")
    elif what == "python":
        import sysconfig
        get = sysconfig.get_config_var
        monkeypatch.setattr(sysconfig, "get_config_var", lambda k: "cpython-399" if k == "SOABI" else get(k))
    else:
        b.BINDING.unlink()
    assert b.binding_needs_build()
    if what in ("torch", "python"):
        assert not b.binding_matches(b.BINDING)         # nor is it loaded
    seen = _compiler(monkeypatch, 0)
    assert b.build() == "library"
    assert any(b.binding_stamp() in arg for arg in seen[0]) and b.BINDING.read_bytes() == b"new"


def test_library_is_built_without_a_compiler_of_the_binding(b, monkeypatch):
    def missing(*a, **kw):
        raise FileNotFoundError("g++")
    monkeypatch.setattr(subprocess, "Popen", missing)
    with pytest.warns(UserWarning, match="g\\+\\+"):
        assert b.build(force=True) == "library"
    assert b.BINDING.exists()                           # it is that of these sources and this torch
    os.utime(b.BINDING, (500, 500))
    with pytest.warns(UserWarning, match="not built"):
        assert b.build() == "library"
    assert not b.BINDING.exists()                       # a stale one does not stay


def test_library_is_built_when_the_binding_does_not_compile(b, monkeypatch):
    _compiler(monkeypatch, 1)
    os.utime(b.BINDING, (500, 500))
    with pytest.warns(UserWarning, match="no such header"):
        assert b.build() == "library"
    assert not b.BINDING.exists()


def test_the_library_error_is_the_one_that_is_raised(b, monkeypatch):
    def broken(force, verbose):
        raise RuntimeError("nvcc failed")
    monkeypatch.setattr(b, "_build_library", broken)
    _compiler(monkeypatch, 1)
    with pytest.warns(UserWarning), pytest.raises(RuntimeError, match="nvcc failed"):
        b.build(force=True)


def test_the_loaded_binding_is_of_this_torch():
    a8, build = load_pkg("attention_kv8"), load_pkg("build")
    if a8._b2torch is not None:
        assert a8._b2torch.stamp == build.binding_stamp()
