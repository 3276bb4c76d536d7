"""Every build compiles every source with the flags of now, whatever objects are there."""
import glob
import os
import subprocess

import __graft_entry__ as entry


def test_every_source_is_compiled_again(monkeypatch):
    compiled, linked = [], []
    monkeypatch.setattr(subprocess, "call", lambda cmd, cwd=None: compiled.append(cmd) or 0)
    monkeypatch.setattr(subprocess, "check_call", lambda cmd, cwd=None: linked.append(cmd) or 0)
    entry._compile_library()
    sources = sorted(glob.glob(os.path.join(entry.PKG, "csrc", "*.hip")))
    assert sorted(c[c.index("-c") + 1] for c in compiled) == sources
    assert all("--offload-arch=gfx950" in c and "-packed-fp32-ops" in c for c in compiled)
    assert len(linked) == 1 and sum(x.endswith(".o") for x in linked[0]) == len(sources)


def test_a_source_that_does_not_compile_is_an_error(monkeypatch):
    linked = []
    monkeypatch.setattr(subprocess, "call", lambda cmd, cwd=None: 1)
    monkeypatch.setattr(subprocess, "check_call", lambda cmd, cwd=None: linked.append(cmd) or 0)
    try:
        entry._compile_library()
    except RuntimeError:
        assert not linked
    else:
        raise AssertionError("no error")
