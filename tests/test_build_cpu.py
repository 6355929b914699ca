"""CPU tests of the library's makefile with a stand-in compiler: every output is made of objects compiled with its own flags."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pgmuvi_amd", "csrc")

# -c: the "object" holds the whole command; else: the "library" is its objects, one after the other.  Every compilation is counted
STAND_IN = """#!/bin/sh
out=; objects=; compile=0; line="$*"
while [ $# -gt 0 ]; do
  case "$1" in -o) out="$2"; shift;; -c) compile=1;; *.o) objects="$objects $1";; esac
  shift
done
if [ $compile = 1 ]; then echo "$line" > "$out"; echo x >> "$COUNT"; else cat $objects > "$out"; fi
"""


@pytest.fixture()
def tree(tmp_path):
    src = tmp_path / "pkg" / "csrc"
    src.mkdir(parents=True)
    (tmp_path / "include").mkdir()
    (tmp_path / "include" / "pgmuvi_hip.h").write_text("")
    for name in os.listdir(CSRC):
        if name.endswith((".hip", ".h", ".inc")):
            (src / name).write_text("")
    shutil.copy(os.path.join(CSRC, "Makefile"), src)
    cc = tmp_path / "cc"
    cc.write_text(STAND_IN)
    cc.chmod(0o755)
    count = tmp_path / "count"

    def make(*args):
        count.write_text("")
        subprocess.run(["make", "-C", str(src), f"HIPCC={cc}", *args], check=True, env=dict(os.environ, COUNT=str(count)), capture_output=True)
        return len(count.read_text().split())

    make.dir = tmp_path
    make.sources = sum(name.endswith(".hip") for name in os.listdir(CSRC))
    return make


def test_a_variant_of_the_same_name_has_objects_of_its_own(tree):
    product, variant = tree.dir / "pkg" / "libpgmuvi_hip.so", tree.dir / "variants" / "foo" / "libpgmuvi_hip.so"
    variant.parent.mkdir(parents=True)
    assert tree(f"OUT={variant}", "EXTRA=-DFOO") == tree.sources
    assert tree() == tree.sources                                # (nothing of the variant's is linked into the product)
    assert "-DFOO" not in product.read_text() and variant.read_text().count("-DFOO") == tree.sources
    assert tree() == 0 and tree(f"OUT={variant}", "EXTRA=-DFOO") == 0


def test_other_flags_for_the_same_output_compile_again(tree):
    product = tree.dir / "pkg" / "libpgmuvi_hip.so"
    assert tree() == tree.sources
    assert tree("EXTRA=-DNAME='\"a b\"'") == tree.sources and "-DNAME" in product.read_text()
    assert tree() == tree.sources and "-DNAME" not in product.read_text()
    assert tree("-B") == tree.sources                            # (always everything)


def test_a_changed_header_or_source_compiles_again(tree):
    assert tree() == tree.sources and tree() == 0
    later = os.path.getmtime(tree.dir / "pkg" / "libpgmuvi_hip.so") + 5
    os.utime(tree.dir / "pkg" / "csrc" / "pgm_ls.hip", (later, later))
    assert tree() >= 1
    os.utime(tree.dir / "include" / "pgmuvi_hip.h", (later + 5, later + 5))
    assert tree() == tree.sources


def test_a_copy_elsewhere_is_built_by_the_same_commands(tree, tmp_path):
    tree()
    copy = tmp_path / "elsewhere" / "deeper"
    shutil.copytree(tree.dir / "pkg", copy / "pkg", ignore=shutil.ignore_patterns("build", "*.so"))
    shutil.copytree(tree.dir / "include", copy / "include")
    subprocess.run(["make", "-C", str(copy / "pkg" / "csrc"), f"HIPCC={tree.dir / 'cc'}"], check=True, env=dict(os.environ, COUNT=os.devnull), capture_output=True)
    assert (copy / "pkg" / "libpgmuvi_hip.so").read_text() == (tree.dir / "pkg" / "libpgmuvi_hip.so").read_text()
