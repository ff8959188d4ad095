"""Scratch buffers that another call replaces between a call's look-up and its launch."""

from __future__ import annotations

import gc
import threading
import weakref

import pytest
import torch

from dominusultra_b200 import _lib, dominus_ultra_decode_paged, paged, precompute_rope_cos_sin

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
