"""Scratch buffers of calls from several threads (no GPU: the allocations are faked on the CPU)."""

from __future__ import annotations

import gc
import weakref

import torch

from dominusultra_b200 import attention, paged


class _OnCpu:
    """torch, with devices and streams that are not there."""

    def __init__(self):
        self.cuda = type("cuda", (), {"is_current_stream_capturing": staticmethod(lambda: False)})

    def __getattr__(self, name):
        return getattr(torch, name)

    @staticmethod
    def device(*_):
        return torch.device("cpu")


def _alive(ref):
    gc.collect()
    return ref() is not None


def test_paged_scratch_outlives_its_replacement(monkeypatch):
    """A call has its scratch, another thread's call on the stream needs a larger one before the first
    is launched: the first one's buffers stay until it lets go of them."""
    monkeypatch.setattr(paged, "torch", _OnCpu())
    monkeypatch.setattr(paged, "_SCRATCH", {})
    monkeypatch.setattr(paged, "_SLABS", {})
    first = paged._decode_scratch(1000, 0, 7)
    ws, tickets = (weakref.ref(t) for t in (paged._SCRATCH[0, 7][4], paged._SCRATCH[0, 7][3]))
    assert first[1] == ws().data_ptr() and first[0] == tickets().data_ptr()
    second = paged._decode_scratch(5000, 0, 7)
    assert second[1] != first[1] and second[0] == first[0]
    assert _alive(ws) and _alive(tickets)
    del first
    assert not _alive(ws) and _alive(tickets)


def test_workspace_outlives_its_replacement(monkeypatch):
    monkeypatch.setattr(attention, "torch", _OnCpu())
    monkeypatch.setattr(attention, "_WORKSPACES", {})
    cpu = torch.device("cpu")
    first = attention._cached_workspace("prefill", 3 << 20, cpu, 7)
    buf = weakref.ref(first[2])
    assert first[:2] == (buf().data_ptr(), 3 << 20)
    second = attention._cached_workspace("prefill", 4 << 20, cpu, 7)
    assert second[1] == 6 << 20 and second[0] != first[0]
    assert _alive(buf)
    del first
    assert not _alive(buf)
    assert attention._cached_workspace("prefill", 0, cpu, 7) == (0, 0, None)


def test_workspace_of_a_capture_is_never_dropped(monkeypatch):
    fake = _OnCpu()
    fake.cuda.is_current_stream_capturing = staticmethod(lambda: True)
    monkeypatch.setattr(attention, "torch", fake)
    monkeypatch.setattr(attention, "_WORKSPACES", {})
    monkeypatch.setattr(attention, "_RETIRED", [])
    cpu = torch.device("cpu")
    first = attention._cached_workspace("decode", 3 << 20, cpu, 7)
    buf = weakref.ref(first[2])
    attention._cached_workspace("decode", 4 << 20, cpu, 7)
    del first
    assert _alive(buf)
