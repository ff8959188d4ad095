"""What the paged extension's Python call keeps of its workspaces' sizes (no GPU)."""

from __future__ import annotations

from dominusultra_b200 import _lib, paged_extend


def test_sizes_are_the_librarys_and_few(monkeypatch):
    monkeypatch.setattr(paged_extend, "_WS_SIZES", {})
    lib = _lib.load()
    for D in (16, 32, 64, 128, 256):
        for Hq, Hkv in ((1, 1), (32, 8), (64, 8), (12, 4)):
            for T in (1, 2, 15, 16, 17, 31, 32, 33, 42, 43, 127, 128, 129, 777, 4096):
                for B, block, width in ((1, 16, 7), (64, 128, 300)):
                    args = (B, Hq, Hkv, T, D, block, width)
                    assert paged_extend._workspace_size(*args, 0) == lib.du_extend_paged_workspace_size(*args) > 0
    assert len(paged_extend._WS_SIZES) <= 10


def test_sizes_that_are_refused_are_not_kept(monkeypatch):
    monkeypatch.setattr(paged_extend, "_WS_SIZES", {})
    assert paged_extend._workspace_size(1, 5, 2, 3, 64, 16, 4, 0) == 0  # (heads that do not divide)
    assert paged_extend._workspace_size(1, 4, 2, 3, 64, 16, 4, 0) > 0
