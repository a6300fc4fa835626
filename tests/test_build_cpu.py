"""The build: what is compiled is compiled again when what compiles it has changed."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "muzero_amd", "csrc")


@pytest.fixture
def tree(tmp_path):
    """A copy of the sources with every target in place and up to date, as empty files."""
    csrc = tmp_path / "muzero_amd" / "csrc"
    csrc.mkdir(parents=True)
    (tmp_path / "include").mkdir()
    shutil.copy(os.path.join(CSRC, "..", "..", "include", "muzero_amd.h"), tmp_path / "include")
    for name in os.listdir(CSRC):
        if name == "Makefile" or name.endswith((".hip", ".h", ".cpp")):
            shutil.copy(os.path.join(CSRC, name), csrc)
    compiled(csrc)                                              # writes flags.stamp
    objects = sorted(n[:-4] + ".o" for n in os.listdir(csrc) if n.endswith(".hip"))
    for name in objects + ["libmuzero_amd.so", "../_blocks.so"]:
        (csrc / name).touch()
    return csrc, objects


def compiled(csrc, *args):
    """The files that make would write."""
    out = subprocess.run(["make", "-n", "-C", str(csrc), *args], check=True, capture_output=True, text=True).stdout
    return {w[w.index("-o") + 1] for w in (line.split() for line in out.splitlines()) if "-o" in w}


def test_nothing_is_compiled_twice(tree):
    assert compiled(tree[0]) == set()


def test_a_changed_makefile_compiles_everything(tree):
    csrc, objects = tree
    os.utime(csrc / "Makefile", (2 ** 31, 2 ** 31))
    assert compiled(csrc) == set(objects) | {"libmuzero_amd.so", "../_blocks.so"}


def test_changed_flags_compile_everything(tree):
    csrc, objects = tree
    past = 2 ** 30
    for name in os.listdir(csrc):                               # mtimes are coarse: what is there is old
        os.utime(csrc / name, (past, past))
    os.utime(csrc.parent.parent / "include" / "muzero_amd.h", (past, past))
    assert compiled(csrc) == set()
    assert compiled(csrc, "CXXFLAGS=-O3 --offload-arch=gfx950") >= set(objects) | {"libmuzero_amd.so"}
