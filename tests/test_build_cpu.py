"""CPU: when the build compiles an object anew."""
import os
import stat

import pytest


@pytest.fixture
def sandbox(tmp_path, monkeypatch):
    """pdae_amd.build on two sources of its own with a compiler that writes its command line into a log."""
    from pdae_amd import build as B
    csrc, lib, log = tmp_path / "csrc", tmp_path / "lib", tmp_path / "log"
    csrc.mkdir()
    for n in ("a.hip", "b.hip"):
        (csrc / n).write_text("// " + n)
    cc = tmp_path / "cc"
    cc.write_text(f"#!/bin/sh\necho \"$@\" >> {log}\nwhile [ $# -gt 1 ]; do if [ \"$1\" = -o ]; then : > \"$2\"; fi; shift; done\n")
    cc.chmod(cc.stat().st_mode | stat.S_IEXEC)
    for k, v in dict(CSRC=str(csrc), LIBDIR=str(lib), LIB=str(lib / "l.so"), SOURCES=["a.hip", "b.hip"], HIPCC=str(cc), FLAGS=["-O3"], EXTRA_FLAGS={}, HAZARD_SCAN=[]).items():
        monkeypatch.setattr(B, k, v)

    def run(**k):
        open(log, "w").close()
        B.build_library(verbose=False, **k)
        return sorted(w for line in open(log) for w in (line.split() if " -c " in f" {line}" else ["link"]) if w.endswith(".hip") or w == "link")
    names = lambda got: [os.path.basename(g) for g in got]
    return B, lambda **k: names(run(**k)), monkeypatch


def test_changed_flags_compile_an_object_anew(sandbox):
    """Flags decide what the kernels compute (no packed fp32 arithmetic, the form of the matrix instructions): an object of other flags is stale."""
    B, build, patch = sandbox
    assert build() == ["a.hip", "b.hip", "link"] and build() == []
    patch.setattr(B, "EXTRA_FLAGS", {"b.hip": ["-x"]})
    assert build() == ["b.hip", "link"] and build() == []
    patch.setattr(B, "FLAGS", ["-O2"])
    assert build() == ["a.hip", "b.hip", "link"] and build() == []
    assert build(force=True) == ["a.hip", "b.hip", "link"]
    os.remove(os.path.join(B.LIBDIR, "a.o"))
    assert build() == ["a.hip", "link"]
    os.utime(os.path.join(B.CSRC, "a.hip"), (2 ** 31 - 1,) * 2)
    assert build() == ["a.hip", "link"]


def test_the_entry_point_compiles_every_source_every_time(monkeypatch):
    import __graft_entry__ as entry
    from pdae_amd import build as B
    asked = []
    monkeypatch.setattr(B, "build_library", lambda **k: asked.append(k) or B.LIB)
    entry.build()
    assert asked == [dict(force=True, verbose=True)]
