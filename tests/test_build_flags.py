"""What makes a build stale, with a compiler that only writes down what it is asked for."""
import os
import stat
import sys

import pytest

from models_amd import build

HIPCC = f"""#!{sys.executable}
import sys, pathlib
a = sys.argv[1:]
here = pathlib.Path(__file__).resolve().parent
if a == ["--version"]:
    print((here / "version").read_text())
    sys.exit(0)
with open(here / "calls", "a") as f:
    f.write(("link" if "-shared" in a else "compile " + pathlib.Path(a[a.index("-c") + 1]).name) + "\\n")
out = pathlib.Path(a[a.index("-o") + 1])
ids = [v.split("0x")[1] for v in a if v.startswith("-Wl,--build-id=")]
out.write_bytes(b"\\x7fELF" + b"".join(bytes.fromhex(i) for i in ids))
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    csrc = tmp_path / "models_amd" / "csrc"
    csrc.mkdir(parents=True)
    (tmp_path / "include").mkdir()
    for p in (csrc / "one.hip", csrc / "two.hip", csrc / "common.h", tmp_path / "include" / "merlin_hip.h"):
        p.write_text(p.name)
        os.utime(p, (1, 1))
    cc = tmp_path / "hipcc"
    cc.write_text(HIPCC)
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    (tmp_path / "version").write_text("1.0")
    monkeypatch.setattr(build, "CSRC", csrc)
    monkeypatch.setattr(build, "LIB", csrc / "libmerlin_hip.so")
    monkeypatch.setattr(build, "_hipcc", lambda: str(cc))
    monkeypatch.delenv("MH_LAB", raising=False)

    def calls(*a, **k):
        log = tmp_path / "calls"
        log.write_text("")
        build.build(*a, **k)
        return sorted(log.read_text().split("\n"))[1:]

    return tmp_path, calls


ALL = ["compile one.hip", "compile two.hip", "link"]


def test_nothing_is_compiled_twice(tree):
    _, calls = tree
    assert calls() == ALL and not build.needs_build() and calls() == []


def test_force_compiles_everything(tree):
    _, calls = tree
    calls()
    assert calls(force=True) == ALL


def test_a_changed_source_is_compiled(tree):
    top, calls = tree
    calls()
    os.utime(top / "models_amd" / "csrc" / "two.hip")
    t = os.stat(build.LIB).st_mtime - 1
    os.utime(build.LIB, (t, t))
    for o in build.CSRC.glob("*.o"):
        os.utime(o, (t, t))
    assert build.needs_build() and calls() == ["compile two.hip", "link"]


def test_other_flags_compile_everything(tree, monkeypatch):
    _, calls = tree
    calls()
    before = build.source_hash()
    monkeypatch.setattr(build, "FLAGS", [*build.FLAGS, "-DSOMETHING"])
    assert build.needs_build() and build.source_hash() != before
    assert calls() == ALL and not build.needs_build()
    assert len(list(build.CSRC.glob("*.o"))) == 2  # none of the other flags' is left


def test_lab_builds_and_shipped_ones_are_kept_apart(tree, monkeypatch):
    _, calls = tree
    calls()
    monkeypatch.setenv("MH_LAB", "1")
    assert build.needs_build() and calls() == ALL and not build.needs_build()
    monkeypatch.delenv("MH_LAB")
    assert build.needs_build() and calls() == ALL


def test_objects_of_another_compiler_are_not_linked(tree):
    top, calls = tree
    calls()
    (top / "version").write_text("2.0")
    t = os.stat(build.LIB).st_mtime
    os.utime(top / "include" / "merlin_hip.h", (t + 1, t + 1))
    assert build.needs_build()
    os.utime(top / "include" / "merlin_hip.h", (1, 1))
    build.LIB.unlink()
    assert calls() == ALL


def test_a_library_that_names_no_flags_is_stale(tree):
    _, calls = tree
    calls()
    build.LIB.write_bytes(b"\x7fELF")
    assert build.needs_build()
    build.LIB.write_bytes(b"")
    assert build.needs_build()
