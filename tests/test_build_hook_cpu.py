"""build() of the driver hooks: the reference's own libraries are compiled where its sources are, not where a folder of its name is."""
import os

import pytest

import __graft_entry__ as entry


@pytest.mark.parametrize("sources", [False, True])
def test_the_reference_is_compiled_only_from_its_sources(monkeypatch, sources):
    import fusedmm_amd.build
    asked = []
    isfile, isdir = os.path.isfile, os.path.isdir
    monkeypatch.setattr(fusedmm_amd.build, "build_all", lambda **kw: asked.append("all"))
    monkeypatch.setattr(entry.subprocess, "check_call", lambda cmd, **kw: asked.append(cmd))
    monkeypatch.setattr(os.path, "isdir", lambda p: True if p == "/root/reference" else isdir(p))
    monkeypatch.setattr(os.path, "isfile", lambda p: sources if p.startswith("/root/reference/") else isfile(p))
    entry.build()
    makes = [c for c in asked if c[0] == "make"]
    assert asked[0] == "all" and any(c[-1] == "all" for c in makes)
    assert any(c[-1] == "ref" for c in makes) == sources
