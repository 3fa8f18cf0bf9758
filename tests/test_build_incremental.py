"""rt_pose_amd.build compiles again what another command made: with a stand-in for hipcc that notes its arguments."""
import os

import pytest

HIPCC = """#!/bin/sh
echo "$@" >> %s
for last; do :; done
out=; prev=
for a; do if [ "$prev" = -o ]; then out=$a; fi; prev=$a; done
if [ -e %s ]; then exit 1; fi
echo made > "$out"
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    from rt_pose_amd import build as b
    for d in ("csrc", "lib"):
        (tmp_path / d).mkdir()
    for f in ("one.hip", "two.hip", "common.h"):
        (tmp_path / "csrc" / f).write_text("x")
        os.utime(tmp_path / "csrc" / f, (1, 1))
    hipcc = tmp_path / "hipcc"
    hipcc.write_text(HIPCC % (tmp_path / "log", tmp_path / "fail"))
    hipcc.chmod(0o755)
    for name, value in (("CSRC", tmp_path / "csrc"), ("OBJ", tmp_path / "lib" / "obj"), ("LIB", tmp_path / "lib" / "x.so"), ("HIPCC", hipcc)):
        monkeypatch.setattr(b, name, str(value))
    monkeypatch.setattr(b, "_deps_mtime", lambda: os.path.getmtime(tmp_path / "csrc" / "common.h"))

    def build(**k):
        log = tmp_path / "log"
        if log.exists():
            log.unlink()
        b.build(verbose=False, **k)
        lines = log.read_text().splitlines() if log.exists() else []
        return ["link" if "-shared" in line else line.split(" -c ")[1].split()[0].split("/")[-1] for line in lines]
    return tmp_path, monkeypatch, b, build


def test_only_what_changed_is_compiled(tree):
    path, _, _, build = tree
    assert sorted(build()) == ["link", "one.hip", "two.hip"] and build() == []
    for made in (path / "lib" / "obj" / "one.o", path / "lib" / "obj" / "two.o", path / "lib" / "x.so"):
        os.utime(made, (100, 100))
    assert build() == []
    os.utime(path / "csrc" / "two.hip", (200, 200))
    assert build() == ["two.hip", "link"] and build() == []
    assert sorted(build(force=True)) == ["link", "one.hip", "two.hip"]


def test_other_flags_and_another_compiler_compile_everything(tree):
    path, monkeypatch, b, build = tree
    build()
    monkeypatch.setattr(b, "FLAGS", [*b.FLAGS, "-DOTHER"])
    assert sorted(build()) == ["link", "one.hip", "two.hip"] and build() == []
    os.utime(path / "hipcc", (5, 5))
    assert sorted(build()) == ["link", "one.hip", "two.hip"] and build() == []


def test_objects_of_an_unknown_command_are_not_linked(tree):
    """What an earlier release, or a build that was broken off, has left."""
    path, _, _, build = tree
    build()
    os.remove(path / "lib" / "obj" / "one.o.cmd")
    assert build() == ["one.hip", "link"]


def test_a_build_that_failed_is_not_up_to_date(tree):
    path, _, _, build = tree
    build()
    (path / "fail").write_text("")
    os.remove(path / "lib" / "x.so.cmd")
    for _ in range(2):
        with pytest.raises(RuntimeError):
            build()
    (path / "fail").unlink()
    assert build() == ["link"] and build() == []
