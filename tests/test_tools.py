"""The tools that build variants of the library (tools/sweep.py, tools/phase_timing_full.py): a variant has every symbol that the Python mirror binds when it loads it."""
import os
import runpy
import subprocess
import sys

import pytest

import tha4_amd  # noqa: F401
from tha4_amd import _build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Done:
    returncode = 0

    def communicate(self):
        return "", ""


@pytest.fixture
def commands(monkeypatch, tmp_path):
    """Commands that a tool would run, instead of running them (a variant compiles for minutes)."""
    seen = []
    monkeypatch.setattr(subprocess, "Popen", lambda cmd, **kw: seen.append(cmd) or Done())
    monkeypatch.setattr(subprocess, "run", lambda cmd, **kw: seen.append(cmd) or Done())
    return seen


@pytest.mark.parametrize("tool,more", [("sweep.py", {"THA4_SWEEP_VARIANTS": "default,stamps,hook"}), ("phase_timing_full.py", {})])
def test_variants_are_built_from_every_source(tool, more, commands, monkeypatch):
    for k, v in more.items():
        monkeypatch.setenv(k, v)
    monkeypatch.setattr(sys, "argv", [tool, "build"])
    try:
        runpy.run_path(os.path.join(ROOT, "tools", tool), run_name="__main__")
    except SystemExit as e:
        assert not e.code
    builds = [c for c in commands if "-shared" in c]
    assert builds
    for c in builds:
        assert {os.path.basename(a) for a in c if a.endswith(".hip")} == set(_build.SOURCES)


def test_build_compiles_every_piece_whenever_it_is_called(monkeypatch):
    """A library that is there already says nothing about the sources that are there now."""
    import torch  # noqa: F401  (loaded before ctypes is replaced)
    import __graft_entry__ as entry
    asked = []
    for module, names in ((_build, ("build_native", "build_forced_wait_twin")), (entry, ("build_emulator", "build_emulator_full", "build_ops_device"))):
        for name in names:
            monkeypatch.setattr(module, name, lambda force=False, name=name: asked.append((name, force)) or _build.LIB)
    monkeypatch.setattr("ctypes.CDLL", lambda path: type("Lib", (), {"__getattr__": lambda self, n: n})())
    entry.build()
    assert sorted(asked) == sorted((n, True) for n in ("build_native", "build_forced_wait_twin", "build_emulator", "build_emulator_full", "build_ops_device"))
