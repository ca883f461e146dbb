"""The build of the serving operators' extension module, its compiler replaced."""
import json
import os
import sys
import types

import pytest

from ennx_b200 import _abi, build


class Compiler:
    """Stands in for subprocess.run: writes the output file, or fails."""

    def __init__(self):
        self.calls, self.fails = [], False

    def __call__(self, cmd, **_):
        self.calls.append(cmd)
        out = cmd[cmd.index("-o") + 1]
        with open(out, "w") as f:
            f.write(f"build {len(self.calls)}")
        return types.SimpleNamespace(returncode=int(self.fails), stdout="", stderr="no")


@pytest.fixture
def compiler(tmp_path, monkeypatch):
    c = Compiler()
    monkeypatch.setattr(build, "BINDINGS", tmp_path / "module.so")
    monkeypatch.setattr(build.subprocess, "run", c)
    return c


def test_without_torch_only_the_module_is_left_out(compiler, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)  # an import raises
    build._build_bindings()
    assert not compiler.calls and "no torch" in capsys.readouterr().err


def test_without_headers_only_the_module_is_left_out(compiler, tmp_path, monkeypatch, capsys):
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(torch, "__file__", str(tmp_path / "torch" / "__init__.py"))
    build._build_bindings()
    assert not compiler.calls and "no C++ headers" in capsys.readouterr().err


def test_a_failing_compiler_is_an_error(compiler):
    pytest.importorskip("torch")
    compiler.fails = True
    with pytest.raises(RuntimeError, match="bindings.cpp"):
        build._build_bindings()
    assert not build.BINDINGS.exists()


def test_the_module_is_rebuilt_when_what_it_was_built_for_changes(compiler, monkeypatch):
    torch = pytest.importorskip("torch")

    def builds():
        before = len(compiler.calls)
        build._build_bindings()
        return len(compiler.calls) - before

    assert builds() == 1 and builds() == 0
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "9.9.9")
        assert builds() == 1 and builds() == 0
    assert builds() == 1  # back
    with monkeypatch.context() as m:
        m.setattr(build.sysconfig, "get_config_var", lambda _: "other-python")
        assert builds() == 1
    with monkeypatch.context() as m:
        m.setenv("CXX", "another++")
        assert builds() == 1
    assert builds() == 1
    os.utime(build.BINDINGS, (1, 1))  # older than its source
    assert builds() == 1 and builds() == 0
    build.BINDINGS.with_suffix(".key").unlink()  # of an unknown origin
    assert builds() == 1


def test_a_failed_build_leaves_the_module_that_was_there_but_not_as_up_to_date(compiler, monkeypatch):
    pytest.importorskip("torch")
    build._build_bindings()
    was = build.BINDINGS.read_text()
    os.utime(build.BINDINGS, (1, 1))
    compiler.fails = True
    for _ in range(2):
        with pytest.raises(RuntimeError):
            build._build_bindings()
        assert build.BINDINGS.read_text() == was and os.listdir(build.BINDINGS.parent) == [build.BINDINGS.name]
    compiler.fails = False
    build._build_bindings()
    assert build.BINDINGS.read_text() != was


@pytest.mark.parametrize("what", ["torch", "python"])
def test_a_module_built_for_another_torch_or_python_is_not_loaded(what, tmp_path, monkeypatch):
    pytest.importorskip("torch")
    (tmp_path / "ennx_b200_serving.so").write_bytes(b"never read")
    (tmp_path / "ennx_b200_serving.key").write_text(json.dumps({**build.bindings_key(), what: "another"}))
    monkeypatch.setattr(_abi, "LIB_PATH", tmp_path / "libennx_b200.so")
    monkeypatch.setattr(_abi, "_serving", None)
    with pytest.raises(_abi.EnnxB200Error, match=f"built for {what} another"):
        _abi.serving()
