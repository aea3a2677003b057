"""pratchya_amd.build where torch is missing builds the library alone, as a host of the
C ABI needs it; with torch the binding too, and a failure of either is an error."""
import sys

import pytest

from pratchya_amd import build as B


@pytest.fixture
def steps(monkeypatch, tmp_path):
    """The compilers' command lines; each writes its output file."""
    ran = []

    def run(cmd):
        ran.append(cmd)
        out = cmd[cmd.index("-o") + 1]
        open(out, "w").close()
        return ""
    monkeypatch.setattr(B, "_run", run)
    monkeypatch.setattr(B, "PKG", tmp_path)
    monkeypatch.setattr(B, "LIB", tmp_path / "libpratchya_fp8.so")
    monkeypatch.setattr(B, "ROW_OPS", tmp_path / "_row_ops.so")
    return ran


def test_without_torch(steps, monkeypatch, capsys):
    B.ROW_OPS.write_text("older")
    monkeypatch.setitem(sys.modules, "torch", None)      # import torch: ImportError
    monkeypatch.setattr("importlib.util.find_spec", lambda name, *a: None)
    assert B.build() == B.LIB and B.LIB.exists()
    assert not B.ROW_OPS.exists() and "torch" in capsys.readouterr().err
    assert not any("row_ops.cpp" in part for cmd in steps for part in cmd)


def test_with_torch(steps):
    assert B.build() == B.LIB and B.LIB.exists() and B.ROW_OPS.exists()
    assert any("row_ops.cpp" in part for part in steps[-1])


def test_errors(steps, monkeypatch):
    run = B._run

    def fails(cmd):
        if any("row_ops.cpp" in part for part in cmd):
            raise RuntimeError("build failed")
        return run(cmd)
    monkeypatch.setattr(B, "_run", fails)
    with pytest.raises(RuntimeError, match="build failed"):
        B.build()
