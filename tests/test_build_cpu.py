"""The library's build stands by itself: torch, which the Python module of the MX operators is compiled against, is not
needed for it, and trouble with that module comes after the library is there."""
import os
import sys

import pytest

from ptwm_amd import build as B


@pytest.fixture
def small(monkeypatch, tmp_path):
    """A build of one source, away from the tree."""
    monkeypatch.setattr(B, "SOURCES", ["xxh64_host.cpp"])
    for name in ("OBJ", "LIB", "MX"):
        monkeypatch.setattr(B, name, str(tmp_path / name.lower()))
    return tmp_path


def test_without_torch(small, monkeypatch):
    monkeypatch.setitem(sys.modules, "torch", None)
    (small / "mx").write_bytes(b"of an earlier build")
    assert B.build() == str(small / "lib")
    assert os.path.getsize(small / "lib") > 0
    assert not (small / "mx").exists()


def test_the_library_is_linked_before_the_module(small, monkeypatch):
    pytest.importorskip("torch")

    def broken():
        raise RuntimeError("no such header")

    monkeypatch.setattr(B, "_compile_mx", broken)
    with pytest.raises(RuntimeError, match="no such header"):
        B.build()
    assert os.path.getsize(small / "lib") > 0
