"""CPU: what the build script takes over from an earlier build."""
import os
import stat

import pytest

from pufferlib_b200 import build

COMPILER = """#!/bin/sh
# stands in for a compiler: logs its arguments, writes its last argument's text and its own to the file after -o
if [ "$1" = "--version" ]; then cat "{dir}/version"; exit 0; fi
echo "$@" >> "{dir}/log"
while [ $# -gt 0 ]; do if [ "$1" = "-o" ]; then out="$2"; fi; last="$1"; shift; done
echo "part of an object" > "$out"
if grep -q broken "$last"; then exit 1; fi
cat "$last" >> "$out"
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    for name in ("one.cu", "two.cu"):
        (tmp_path / name).write_text(name)
    (tmp_path / "version").write_text("compiler 1")
    script = tmp_path / "cc"
    script.write_text(COMPILER.format(dir=tmp_path))
    script.chmod(script.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setattr(build, "CSRC", str(tmp_path))
    monkeypatch.setattr(build, "OBJ_DIR", str(tmp_path / "build"))

    class Tree:
        def run(self, *flags, force=False, torch_version="1", **kw):
            """The sources compiled by this call."""
            (tmp_path / "log").write_text("")
            self.objects = build._objects(["one.cu", "two.cu"], [], [str(script), *flags], force, False, versions=[torch_version], **kw)
            return [line.split()[-1].split("/")[-1] for line in (tmp_path / "log").read_text().splitlines()]
    t = Tree()
    t.dir = tmp_path
    return t


def later(path):
    """As if written a while after everything else."""
    t = os.path.getmtime(path) + 100
    os.utime(path, (t, t))


def test_objects_are_kept_only_under_the_same_settings(tree):
    both = ["one.cu", "two.cu"]
    assert sorted(tree.run("-O2")) == both
    assert tree.run("-O2") == []
    assert sorted(tree.run("-O3")) == both                       # another command
    assert tree.run("-O3") == []
    assert sorted(tree.run("-O3", torch_version="2")) == both    # other headers
    (tree.dir / "version").write_text("compiler 2")              # another compiler
    assert sorted(tree.run("-O3", torch_version="2")) == both
    assert tree.run("-O3", torch_version="2") == []
    assert sorted(tree.run("-O3", torch_version="2", force=True)) == both


def test_a_changed_source_is_compiled_alone(tree):
    tree.run("-O2")
    (tree.dir / "two.cu").write_text("two, again")
    later(tree.dir / "two.cu")
    assert tree.run("-O2") == ["two.cu"]


def test_flags_that_only_print_leave_no_trace(tree):
    tree.run("-O2")
    assert len(tree.run("-O2", force=True, also=["-Xptxas", "-v"])) == 2
    assert "-Xptxas -v" in (tree.dir / "log").read_text()
    assert tree.run("-O2") == []


def test_no_part_of_an_object_stays_behind(tree):
    (tree.dir / "two.cu").write_text("broken")
    with pytest.raises(Exception):
        tree.run("-O2")
    left = os.listdir(tree.dir / "build")
    assert not any(n.startswith("two.cu") for n in left) and any(n.startswith("one.cu") for n in left)
    (tree.dir / "two.cu").write_text("mended")
    assert tree.run("-O2") == ["two.cu"]
    assert (tree.dir / "build" / os.path.basename(tree.objects[1])).read_text().endswith("mended")
    # a build that is broken off leaves the object of the one before it whole
    (tree.dir / "two.cu").write_text("broken")
    later(tree.dir / "two.cu")
    with pytest.raises(Exception):
        tree.run("-O2")
    assert not any("part" in (tree.dir / "build" / n).read_text() and n.endswith(".o") and "mended" not in
                   (tree.dir / "build" / n).read_text() and n.startswith("two") for n in os.listdir(tree.dir / "build"))


def test_a_library_of_other_settings_is_stale(tree):
    lib = tree.dir / "lib.so"
    assert build._stale(str(lib), [])
    lib.write_text("library")
    assert not build._stale(str(lib), [], "a")       # one that came without a record goes by its age
    build._record(str(lib), "a")
    assert not build._stale(str(lib), [], "a")
    assert build._stale(str(lib), [], "b")
