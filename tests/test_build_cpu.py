"""The build's own bookkeeping, with a stand-in for the compiler."""
import os

import pytest


@pytest.fixture
def tree(tmp_path, monkeypatch):
    "build.py over two sources in an empty directory; the compiler writes its command line into what it makes"
    from transvae_amd import build
    here, csrc, lib = tmp_path / "pkg", tmp_path / "pkg" / "csrc", tmp_path / "pkg" / "lib"
    csrc.mkdir(parents=True)
    (tmp_path / "include").mkdir()
    for f in (csrc / "common.h", csrc / "gemm_common.h", tmp_path / "include" / "tvae_kernels.h", csrc / "a.hip", csrc / "b.hip"):
        f.write_text("")
    cc, log = tmp_path / "cc", tmp_path / "log"
    cc.write_text('#!/bin/sh\nall="$*"\nwhile [ "$1" != -o ]; do shift; done\ncase "$all" in *--fail*) case "$2" in *b.o) exit 1;; esac;; esac\n'
                  'echo "$all" > "$2"\necho "$2" >> %s\n' % log)
    cc.chmod(0o755)
    for name, value in (("HERE", str(here)), ("CSRC", str(csrc)), ("LIBDIR", str(lib)), ("LIB", str(lib / "l.so")), ("SOURCES", ["a.hip", "b.hip"]),
                        ("FLAGS", ["-O3"]), ("_hipcc", lambda: str(cc))):
        monkeypatch.setattr(build, name, value)

    def made():
        "names of what was made since the last call"
        names = [os.path.basename(x) for x in log.read_text().split()] if log.exists() else []
        log.write_text("")
        return sorted(names)
    return build, lib, made, csrc


def test_objects_are_made_once_and_again_for_a_changed_source(tree):
    build, lib, made, csrc = tree
    build.build_lib()
    assert made() == ["a.o", "b.o", "l.so"]
    build.build_lib()
    assert made() == []
    later = os.path.getmtime(lib / "l.so") + 5
    os.utime(csrc / "b.hip", (later, later))
    build.build_lib()
    assert made() == ["b.o", "l.so"]


def test_changed_flags_make_every_object_again(tree, monkeypatch):
    "also where a build with them failed half way and the flags were taken back"
    build, lib, made, _ = tree
    build.build_lib()
    made()
    monkeypatch.setattr(build, "FLAGS", ["-O3", "-new"])
    build.build_lib()
    assert made() == ["a.o", "b.o", "l.so"] and "-new" in (lib / "a.o").read_text()
    build.build_lib()
    assert made() == []
    monkeypatch.setattr(build, "FLAGS", ["-O3", "--fail"])
    with pytest.raises(RuntimeError):
        build.build_lib()
    made()
    monkeypatch.setattr(build, "FLAGS", ["-O3", "-new"])
    build.build_lib()
    assert made() == ["a.o", "b.o", "l.so"] and "--fail" not in (lib / "a.o").read_text()
