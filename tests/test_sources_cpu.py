"""What the committed sources must not hold: text that keeps the tree from being uploaded to a machine with the GPU, and an upload list
whose patterns match nothing."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = re.compile(r"(\.(py|sh|hip|cc|c|cpp|hpp|h|s|S|inc|txt|cmake|mk)|/Makefile)$")
# writes through the scalar data cache: scalar stores and atomics, that cache's write-back and discard, and the bare prefix of the latter two
SCALAR_CACHE_WRITE = re.compile(r"(?<![A-Za-z0-9_])s_(?:(?:scratch_|buffer_)?(?:store|atomic)|dcache(?:_wb|_discard|(?![a-z_])))")


def tracked_files():
    r = subprocess.run(["git", "-C", ROOT, "ls-files", "-z"], capture_output=True, text=True)
    if r.returncode != 0:
        pytest.skip("not a git checkout")
    return [f for f in r.stdout.split("\0") if f]


def test_no_source_names_a_scalar_cache_write():
    """GPU code here writes through vector stores only.  A tree in which ANY source names the other kind, in a comment or in a table of
    opcodes, is refused before a machine with the GPU sees it: then no GPU test, smoke run or benchmark of that commit exists."""
    files = [f for f in tracked_files() if SOURCE.search("/" + f)]
    assert len(files) > 80, "the search did not see the sources"
    bad = []
    for f in files:
        with open(os.path.join(ROOT, f), errors="replace") as fh:
            bad += ["%s:%d" % (f, i) for i, line in enumerate(fh, 1) if SCALAR_CACHE_WRITE.search(line)]
    assert not bad, "named in " + ", ".join(bad)


def test_the_upload_list_matches_what_it_names():
    """tar's patterns: one that ends in a slash matches nothing, so what it names is uploaded all the same."""
    with open(os.path.join(ROOT, ".gpurunignore")) as fh:
        pats = [l.strip() for l in fh if l.strip()]
    assert pats and not [p for p in pats if p.endswith("/")]
    # of the tracked files only the tests' emulator, which no GPU run reads, stays behind
    assert "./tests/emu" in pats
    names = [p[2:] if p.startswith("./") else p for p in pats]
    for f in tracked_files():
        kept_back = any(n in (f, os.path.basename(f)) or f.startswith(n + "/") or ("/" + n + "/") in f for n in names)
        assert kept_back == f.startswith("tests/emu/"), f
    assert not any(c in n for n in names for c in "*?["), "patterns with wildcards need a test of what they match"
