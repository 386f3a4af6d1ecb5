"""Which files a build makes again (no compiler runs: a script that writes its output file and a line about its arguments stands in for it)."""
import os
import stat

import pytest

from uncrtaints_amd import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    src, lib, log = tmp_path / "csrc", tmp_path / "lib", tmp_path / "log"
    src.mkdir()
    for name in ("a.hip", "b.hip", "dev_probes.hip", "common.h"):
        (src / name).write_text(name)
        os.utime(src / name, (1, 1))
    cc = tmp_path / "cc"
    cc.write_text(f'#!/bin/sh\nfor last; do :; done\necho "$@" >> {log}\ncase "$*" in *-DBROKEN*) exit 1;; esac\necho made > "$last"\n')
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("HIPCC", str(cc))
    monkeypatch.setattr(build, "CSRC", str(src))
    monkeypatch.setattr(build, "LIBDIR", str(lib))
    monkeypatch.setattr(build, "LIB", str(lib / "libuncr_hip.so"))
    monkeypatch.setattr(build, "DEV_LIB", str(lib / "libuncr_dev.so"))
    monkeypatch.setattr(build, "FLAGS", ["-O3"])
    monkeypatch.setattr(build, "SOURCES", [("a", [], "a"), ("b", ["-DP=0"], "b_p0"), ("b", ["-DP=1"], "b_p1")])

    def made(**kw):
        """One build -> the names of the files it made"""
        log.write_text("")
        build.build_lib(**kw)
        return sorted(os.path.basename(line.split()[-1]) for line in log.read_text().splitlines())

    return made, src, lib, monkeypatch


ALL = ["a.o", "b_p0.o", "b_p1.o", "libuncr_dev.so", "libuncr_hip.so"]


def test_a_build_makes_what_is_old(tree):
    made, src, lib, _ = tree
    assert made() == ALL and made() == [] and made(force=True) == ALL
    os.utime(src / "a.hip")
    os.utime(lib / "obj" / "a.o", (2, 2))
    assert made() == ["a.o", "libuncr_hip.so"]
    os.utime(lib / "libuncr_hip.so", (2, 2))          # a link that did not happen after the objects were made
    assert made() == ["libuncr_hip.so"]


def test_a_build_makes_again_what_other_flags_made(tree):
    made, _, lib, patch = tree
    assert made() == ALL
    patch.setattr(build, "FLAGS", ["-O3", "-mno-packed"])
    assert made() == ALL and made() == []
    patch.setattr(build, "SOURCES", [("a", [], "a"), ("b", ["-DP=0"], "b_p0"), ("b", ["-DP=2"], "b_p1")])
    assert made() == ["b_p1.o", "libuncr_hip.so"]
    os.remove(lib / "obj" / "a.o.flags")               # built before flags were recorded: not known to be the present ones
    assert made() == ["a.o", "libuncr_hip.so"]


def test_a_failed_build_is_made_again(tree):
    made, _, _, patch = tree
    assert made() == ALL
    good = list(build.SOURCES)
    patch.setattr(build, "SOURCES", good[:1] + [("b", ["-DBROKEN"], "b_p0")])
    with pytest.raises(RuntimeError, match="hipcc failed"):
        made()
    patch.setattr(build, "SOURCES", good)
    assert made() == ["b_p0.o", "libuncr_hip.so"]


def test_the_hash_of_the_sources_covers_the_flags(tree):
    _, src, _, patch = tree
    first = build.source_sha()
    patch.setattr(build, "FLAGS", ["-O2"])
    second = build.source_sha()
    patch.setattr(build, "SOURCES", [("a", ["-DX"], "a")])
    third = build.source_sha()
    (src / "a.hip").write_text("other")
    assert len({first, second, third, build.source_sha()}) == 4
