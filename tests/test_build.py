"""build() of __graft_entry__.py, without compiling anything."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import __graft_entry__ as g  # noqa: E402


@pytest.fixture
def no_compiler(monkeypatch, tmp_path):
    """The commands that build() would run, in place of their effects; a tree of sources of its own."""
    commands = []

    class Process:
        def __init__(self, cmd):
            commands.append(cmd)

        def wait(self, timeout=None):
            return 0

    for sub in ("csrc", "lib", "include"):
        (tmp_path / sub).mkdir()
    (tmp_path / "csrc" / "a.hip").write_text("int a;\n")
    (tmp_path / "csrc" / "b.hpp").write_text("int b;\n")
    (tmp_path / "include" / "nmfx.h").write_text("int c;\n")
    monkeypatch.setattr(subprocess, "Popen", Process)
    monkeypatch.setattr(subprocess, "check_call", lambda cmd, **kw: commands.append(cmd))
    monkeypatch.setattr(g, "ROOT", str(tmp_path))
    monkeypatch.setattr(g, "CSRC", str(tmp_path / "csrc"))
    monkeypatch.setattr(g, "LIBDIR", str(tmp_path / "lib"))
    return commands


def test_build_compiles_with_and_without_force(built, no_compiler):
    for kw in ({}, {"force": True}, {"force": False}):
        no_compiler.clear()
        g.build(**kw)
        assert sum("-c" in cmd for cmd in no_compiler) == 5 and any("-shared" in cmd for cmd in no_compiler)


def test_a_library_of_other_sources_is_noticed(built, no_compiler, tmp_path):
    assert not g.stale()                                  # nothing is recorded: nothing is known
    g.build()
    assert not g.stale()
    for path in ("csrc/a.hip", "csrc/b.hpp", "include/nmfx.h"):
        before = (tmp_path / path).read_text()
        (tmp_path / path).write_text(before + "// changed\n")
        assert g.stale(), path
        (tmp_path / path).write_text(before)
        assert not g.stale()
    (tmp_path / "csrc" / "new.hpp").write_text("int d;\n")
    assert g.stale()
    g.build()
    assert not g.stale()
    (tmp_path / "csrc" / "a.o").write_text("compiled")    # not a source
    assert not g.stale()


def test_a_failed_build_leaves_no_record(built, no_compiler, monkeypatch, tmp_path):
    g.build()
    (tmp_path / "csrc" / "a.hip").write_text("int a2;\n")

    def fails(cmd, **kw):
        raise subprocess.CalledProcessError(1, cmd)

    monkeypatch.setattr(subprocess, "check_call", fails)
    with pytest.raises(subprocess.CalledProcessError):
        g.build()
    assert not (tmp_path / "lib" / g.RECORD).exists()
