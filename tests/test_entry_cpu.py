"""The entry points at the repository's root: what build() compiles, and from what."""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

import __graft_entry__ as entry  # noqa: E402


def commands_of_build(monkeypatch, reference):
    """build()'s compile calls, with the library's own compilation and every child process recorded instead of run."""
    from mallie_amd import build as b
    calls = []
    monkeypatch.setattr(b, "build", lambda **k: calls.append(("library", k)))
    monkeypatch.setattr(entry.subprocess, "run", lambda cmd, **k: calls.append((cmd[-1], k)))
    monkeypatch.setattr(entry, "REFERENCE", str(reference))
    entry.build()
    return calls


def test_build_passes_beside_an_empty_reference_folder(monkeypatch, tmp_path):
    """The reference's sources are optional: a folder without them is as good as none, and must not fail the build."""
    assert [c for c, _ in commands_of_build(monkeypatch, tmp_path)] == ["library", "oracle"]
    assert [c for c, _ in commands_of_build(monkeypatch, tmp_path / "missing")] == ["library", "oracle"]


def test_build_compiles_the_reference_where_its_sources_are(monkeypatch, tmp_path):
    (tmp_path / "render.cc").write_text("")
    calls = commands_of_build(monkeypatch, tmp_path)
    assert [c for c, _ in calls] == ["library", "oracle", "ref"] and calls[2][1]["check"]


def test_build_compiles_the_library_also_where_one_is_built(monkeypatch, tmp_path):
    """build() answers whether the sources compile: a library left by an earlier build must not stand in for them."""
    assert commands_of_build(monkeypatch, tmp_path)[0] == ("library", {"force": True})
