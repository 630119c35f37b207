"""When the built libraries are taken to be out of date."""
import os

import pytest

from instancerefer_amd import _build


@pytest.mark.parametrize("which", ["library", "nodes"])
def test_a_changed_recipe_makes_them_stale(which, tmp_path, monkeypatch):
    """the compiler's flags stand in _build.py: a library older than it may be built with others"""
    built = tmp_path / "built.so"
    built.write_bytes(b"")
    for name in ("SOURCES", "HEADERS", "NODES_SRCS", "NODES_HDRS"):
        monkeypatch.setattr(_build, name, [])
    monkeypatch.setattr(_build, "LIB_PATH" if which == "library" else "NODES_PATH", str(built))
    stale = _build._stale if which == "library" else _build.nodes_stale
    recipe = os.path.getmtime(_build.__file__)
    os.utime(built, (recipe + 10, recipe + 10))
    assert not stale()
    os.utime(built, (recipe - 10, recipe - 10))
    assert stale()
