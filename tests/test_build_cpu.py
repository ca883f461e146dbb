"""The build of the serving operators' extension module, its compiler replaced."""
import subprocess
import sys
import types

import pytest

from ennx_b200 import build


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
    assert subprocess.run is compiler
