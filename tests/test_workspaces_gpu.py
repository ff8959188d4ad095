"""Scratch buffers that another call replaces between a call's look-up and its launch."""

from __future__ import annotations

import gc
import threading
import weakref

import pytest
import torch

from dominusultra_b200 import (
    _lib,
    attention,
    decode_partial,
    dominus_ultra_decode,
    dominus_ultra_decode_kvcache,
    dominus_ultra_decode_paged,
    dominus_ultra_prefill,
    paged,
    precompute_rope_cos_sin,
)

pytestmark = pytest.mark.gpu

DEV = "cuda"


class _Before:
    """The library, with `act` called right before one of its functions."""

    def __init__(self, lib, name, act):
        self._lib, self._name, self._act = lib, name, act

    def __getattr__(self, name):
        f = getattr(self._lib, name)
        if name != self._name:
            return f

        def call(*args):
            self._act()
            return f(*args)

        return call


def _paged_args(n):
    g = torch.Generator(device=DEV).manual_seed(n)
    pages = -(-n // 16)
    k, v = (torch.randn(pages, 2, 16, 64, generator=g, device=DEV).to(torch.float8_e4m3fn) for _ in range(2))
    one = torch.ones(pages, 2, device=DEV)
    cos, sin = precompute_rope_cos_sin(n, 64, DEV, torch.bfloat16)
    q = torch.randn(1, 8, 1, 64, generator=g, device=DEV).bfloat16()
    i32 = dict(dtype=torch.int32, device=DEV)
    return q, k, v, one, one, torch.arange(pages, **i32)[None], torch.tensor([n], **i32), cos, sin


def test_paged_decode_keeps_its_scratch_until_the_launch(cuda_device, monkeypatch):
    args = _paged_args(3000)
    want = dominus_ultra_decode_paged(*args)
    index, stream = torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream
    held = weakref.ref(paged._SCRATCH[index, stream][4])
    seen = []

    def replace():  # what another thread's call with a larger batch does
        paged._grow_scratch(2 * paged._SCRATCH[index, stream][2], index, stream)
        gc.collect()
        seen.append(held() is not None)

    monkeypatch.setattr(paged._lib, "load", lambda lib=_lib.load(): _Before(lib, "du_decode_paged", replace))
    got = dominus_ultra_decode_paged(*args)
    gc.collect()
    assert seen == [True] and held() is None
    assert torch.equal(got, want)


def test_paged_decode_from_threads(cuda_device):
    """Calls of several sizes from four threads on the default stream, with memory that comes and goes."""
    sets = [_paged_args(n) for n in (300, 3000, 9000, 20000)]
    want = [dominus_ultra_decode_paged(*a) for a in sets]
    torch.cuda.synchronize()
    with paged._SLAB_LOCK:
        paged._SCRATCH.clear()
    bad = []

    def work(i):
        for j in range(60):
            junk = torch.full((1 << 18,), float(j), device=DEV)
            got = dominus_ultra_decode_paged(*sets[(i + j) % 4])
            if not torch.equal(got, want[(i + j) % 4]) or not bool((junk == j).all()):
                bad.append((i, j))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    assert _lib.read_status(reset=True)[0] == 0


@pytest.mark.parametrize("name", ["prefill", "decode", "decode_partial", "decode_kvcache"])
def test_calls_keep_their_workspace_until_the_launch(cuda_device, monkeypatch, name):
    B, Hq, Hkv, L, D = 1, 8, 2, 20000, 64
    T = 5000 if name == "prefill" else L
    g = torch.Generator(device=DEV).manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    q, k, v = r(B, Hq, T if name == "prefill" else 1, D), r(B, Hkv, T, D), r(B, Hkv, T, D)
    cos, sin = precompute_rope_cos_sin(T + 1, D, DEV, torch.bfloat16)
    lens = torch.tensor([L], dtype=torch.int32, device=DEV)
    call = {
        "prefill": lambda: dominus_ultra_prefill(q, k, v, cos, sin, Hkv)[0],
        "decode": lambda: dominus_ultra_decode(q, k, v, cos, sin, Hkv),
        "decode_partial": lambda: decode_partial(q, k, v, cos, sin, Hkv, L, 0)[0],
        "decode_kvcache": lambda: dominus_ultra_decode_kvcache(q, k, v, cos, sin, lens, num_kv_heads=Hkv),
    }[name]
    kind = "decode" if name == "decode_partial" else name
    want = call()
    key = (kind, torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream)
    entry = attention._WORKSPACES[key]
    entry[1] = False  # (a capture of an earlier test would keep the buffer)
    held = weakref.ref(entry[0])
    size = entry[0].numel()
    del entry
    seen = []

    def replace():
        attention._cached_workspace(kind, size + 1, q.device, key[2])
        gc.collect()
        seen.append(held() is not None)

    monkeypatch.setattr(attention._lib, "load", lambda lib=_lib.load(): _Before(lib, "du_" + name, replace))
    got = call()
    gc.collect()
    assert seen == [True] and held() is None
    assert torch.equal(got, want)


@pytest.mark.parametrize("slab", ["none yet", "used up"])
def test_captures_without_a_ticket_slab(cuda_device, monkeypatch, slab):
    """A process's first paged decode inside a capture, and captures beyond a slab's tickets: the graph zeroes
    tickets of its own, on every replay."""
    args = _paged_args(9000)
    want = dominus_ultra_decode_paged(*args)
    if slab == "none yet":
        monkeypatch.setattr(paged, "_SLABS", {})
    else:
        index = torch.cuda.current_device()
        monkeypatch.setattr(paged, "_SLABS", {index: [paged._SLABS[index][0], paged._SLAB_WORDS]})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [dominus_ultra_decode_paged(*args) for _ in range(3)]
        outs.append(torch.full_like(outs[0], 3.0))  # (what may take the memory of tickets given back)
        outs.append(dominus_ultra_decode_paged(*args))
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        assert all(torch.equal(o, want) for i, o in enumerate(outs) if i != 3)
    assert _lib.read_status(reset=True)[0] == 0
