"""CPU: the build's bookkeeping, with a compiler that only writes down what it was given."""
import os
import stat

import pytest

from recflex_b200 import build

COMPILER = """#!/bin/sh
# writes the source's text (or, when linking, the objects' text) to the output, as a compiler does: not at once
last=""; out=""; srcs=""
for a in "$@"; do
  if [ "$last" = "-o" ]; then out="$a"; fi
  case "$a" in *.cu|*.o) if [ "$last" != "-o" ]; then srcs="$srcs $a"; fi;; esac
  last="$a"
done
echo begun > "$out"
echo "$out" >> "$LOG"
if [ -e "$BREAK" ]; then exit 9; fi
cat $srcs > "$out"
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    csrc, objects = tmp_path / "csrc", tmp_path / "build"
    csrc.mkdir()
    nvcc = tmp_path / "nvcc"
    nvcc.write_text(COMPILER)
    nvcc.chmod(nvcc.stat().st_mode | stat.S_IXUSR)
    for name in ("a", "b"):
        (csrc / f"{name}.cu").write_text(f'#include "shared.h"\nfirst {name}\n')
    (csrc / "shared.h").write_text("header\n")
    monkeypatch.setenv("LOG", str(tmp_path / "log"))
    monkeypatch.setenv("BREAK", str(tmp_path / "break"))
    monkeypatch.setattr(build, "_nvcc", lambda: str(nvcc))
    monkeypatch.setattr(build, "CSRC", str(csrc))
    monkeypatch.setattr(build, "BUILD_DIR", str(objects))
    monkeypatch.setattr(build, "LIB_PATH", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build, "_units", lambda: [("a.o", "a.cu", []), ("b.o", "b.cu", [])])
    return tmp_path


def library(tree):
    return (tree / "lib.so").read_text()


def test_units_are_rebuilt_by_what_they_are_made_of(tree):
    build.build()
    assert "first a" in library(tree) and "first b" in library(tree)
    (tree / "log").unlink()
    build.build()
    assert not (tree / "log").exists()
    (tree / "csrc" / "b.cu").write_text('#include "shared.h"\nsecond b\n')
    build.build()
    assert "first a" in library(tree) and "second b" in library(tree) and "first b" not in library(tree)
    assert "a.o" not in (tree / "log").read_text()
    (tree / "csrc" / "shared.h").write_text("other header\n")
    (tree / "log").unlink()
    build.build()
    assert "a.o" in (tree / "log").read_text() and "b.o" in (tree / "log").read_text()


def test_a_build_that_broke_off_leaves_nothing_that_looks_finished(tree):
    """A source changed, the compiler broke off in the middle of its output, the source put back and another one changed:
    the broken object is not linked."""
    build.build()
    good = library(tree)
    source = tree / "csrc" / "a.cu"
    first = source.read_text()
    source.write_text("third a\n")
    (tree / "break").touch()
    with pytest.raises(RuntimeError):
        build.build()
    (tree / "break").unlink()
    source.write_text(first)
    (tree / "csrc" / "b.cu").write_text("second b\n")
    build.build()
    assert "first a" in library(tree) and "second b" in library(tree)
    (tree / "csrc" / "b.cu").write_text('#include "shared.h"\nfirst b\n')
    build.build()
    assert library(tree) == good


def test_a_build_that_was_killed_before_it_noted_what_it_built(tree, monkeypatch):
    """The object of the new source is there, the note beside it is of the old one; then the old source comes back."""
    build.build()
    source = tree / "csrc" / "a.cu"
    first = source.read_text()
    source.write_text("third a\n")
    real = open

    def killed(path, mode="r", *args, **kw):
        if "w" in mode and "sha256" in os.path.basename(str(path)):
            raise KeyboardInterrupt
        return real(path, mode, *args, **kw)

    with monkeypatch.context() as m:
        m.setattr("builtins.open", killed)
        with pytest.raises(KeyboardInterrupt):
            build.build(jobs=1)
    source.write_text(first)
    (tree / "csrc" / "b.cu").write_text("second b\n")
    build.build()
    assert "first a" in library(tree) and "second b" in library(tree)


def test_a_link_that_broke_off_is_done_again(tree, monkeypatch):
    build.build()
    good = library(tree)
    source = tree / "csrc" / "a.cu"
    first = source.read_text()
    source.write_text("third a\n")
    compile_one = build._compile

    def then_break(*args):
        compile_one(*args)
        (tree / "break").touch()

    with monkeypatch.context() as m:
        m.setattr(build, "_units", lambda: [("a.o", "a.cu", []), ("b.o", "b.cu", [])])
        m.setattr(build, "_compile", then_break)
        with pytest.raises(RuntimeError):
            build.build(jobs=1)
    (tree / "break").unlink()
    source.write_text(first)
    build.build()
    assert library(tree) == good
    assert not [f for f in os.listdir(tree / "build") if f not in ("a.o", "b.o", "a.o.sha256", "b.o.sha256", "sources.sha256")]


def test_a_note_that_goes_away_while_it_is_read_is_no_note(tree, monkeypatch):
    """Another process takes the notes away when it begins to build."""
    build.build()
    monkeypatch.setattr(build.os.path, "exists", lambda path: True)
    assert build._read(str(tree / "build" / "gone.sha256")) == ""
