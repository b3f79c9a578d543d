"""The library builds where its optional Python module does not: no compiler of the host's, no headers of torch or Python, no torch."""
import importlib.util
import os
import subprocess
import types

import pytest

import __graft_entry__ as entry


@pytest.mark.parametrize("missing", ["headers", "compiler", "torch"])
def test_the_module_is_optional(missing, tmp_path, monkeypatch, capsys):
    entry.build_library()
    mod = entry._load_build_module()
    stale = tmp_path / "_fast.so"
    stale.write_bytes(b"made for another torch")
    os.utime(stale, (0, 0))
    monkeypatch.setattr(mod, "FAST", str(stale))
    real, find = subprocess.run, importlib.util.find_spec

    def run(cmd, **kw):
        if cmd[0] != "g++":
            return real(cmd, **kw)
        if missing == "compiler":
            raise FileNotFoundError("g++")
        return types.SimpleNamespace(returncode=1, stdout="", stderr="Python.h: No such file")
    monkeypatch.setattr(mod.subprocess, "run", run)
    if missing == "torch":
        monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    assert mod.build() == mod.LIB
    assert not stale.exists() and "_fast.so is not built" in capsys.readouterr().err
