"""The first call of an extension or a compaction waits for no copy from the host (no GPU: the allocations are faked)."""

from __future__ import annotations

from dominusultra_b200 import paged
from tests.test_workspaces_cpu import _OnCpu


def test_a_workspace_brings_no_tickets_from_the_host(monkeypatch):
    monkeypatch.setattr(paged, "torch", _OnCpu())
    monkeypatch.setattr(paged, "_SCRATCH", {})
    monkeypatch.setattr(paged, "_SLABS", {})
    ws, keep = paged._workspace(1000, 0, 7)
    assert paged._SLABS == {} and ws == keep[4].data_ptr() and keep[2] >= 1000
    # a decode behind it, on the same stream, gets its slab, and the same scratch
    tickets, same, _ = paged._decode_scratch(1000, 0, 7)
    assert same == ws and tickets == keep[3].data_ptr() and 0 in paged._SLABS
    # larger ones grow it, with tickets or without
    assert paged._workspace(5000, 0, 7)[1][2] >= 5000 and len(paged._SLABS) == 1
