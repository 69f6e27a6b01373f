"""The build entry compiles every source on every call, also where a built library is there."""
import glob
import os
import subprocess
import types

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_build_entry_compiles_every_source(monkeypatch):
    import __graft_entry__ as entry
    calls = []

    def run(cmd, **kwargs):                                  # (what it would run; the libraries that are there stay as they are)
        calls.append([str(c) for c in cmd])
        return types.SimpleNamespace(returncode=0, stderr="", stdout="")

    monkeypatch.setattr(subprocess, "run", run)
    entry.build()
    compiled = {os.path.basename(c[c.index("-c") + 1]) for c in calls if "-c" in c}
    sources = {os.path.basename(p) for p in glob.glob(os.path.join(ROOT, "mb-vae-dti_amd", "csrc", "*.hip"))}
    assert compiled == sources
    assert all("--offload-arch=gfx950" in c and "-packed-fp32-ops" in c for c in calls if "-c" in c)
    assert any(c[-1].endswith("host.cpp") or any(a.endswith("host.cpp") for a in c) for c in calls), "the extension module"
    assert any("-shared" in c and any(a.endswith("embedding.o") for a in c) for c in calls), "the library is linked"
