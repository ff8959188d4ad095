"""Paged calls whose inputs come from another stream, a copy or a fork inside a capture. The kernels may start
beside the kernel before them on their stream; what they read has to be there all the same."""

from __future__ import annotations

import pytest
import torch

from dominusultra_b200 import (
    _lib,
    dominus_ultra_decode_paged,
    dominus_ultra_paged_tables,
    dominus_ultra_paged_write,
    precompute_rope_cos_sin,
)

pytestmark = pytest.mark.gpu

DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)
B, HQ, HKV, D, BLOCK, WIDTH = 4, 8, 2, 128, 16, 64


@pytest.fixture(autouse=True)
def _clean_status(cuda_device):
    _lib.read_status(reset=True)
    yield
    assert _lib.read_status(reset=True)[0] == 0, "a test left a device status"


class _Step:
    """Requests of 500 tokens in a paged cache and a step of one more token each."""

    def __init__(self, seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
        n = B * WIDTH
        self.k8, self.v8 = (torch.zeros(n, HKV, BLOCK, D, device=DEV).to(torch.float8_e4m3fn) for _ in range(2))
        self.ks, self.vs = torch.zeros(n, HKV, device=DEV), torch.zeros(n, HKV, device=DEV)
        self.table = torch.full((B, WIDTH), -1, **I32)
        self.ring, self.state = torch.arange(n, **I32), torch.tensor([0, n], **I32)
        self.cos, self.sin = precompute_rope_cos_sin(WIDTH * BLOCK, D, DEV, torch.bfloat16)
        zero = torch.zeros(B, **I32)
        slots, self.lens, self.state = dominus_ultra_paged_tables(self.table, zero, zero + 500, self.ring, self.state, BLOCK, 500)
        self.write(r(B, HKV, 500, D), r(B, HKV, 500, D), slots, zero)
        self.q, self.k, self.v = r(B, HQ, 1, D), r(B, HKV, 1, D), r(B, HKV, 1, D)

    def write(self, k, v, slots, past):
        dominus_ultra_paged_write(k, v, self.k8, self.v8, self.ks, self.vs, slots, past, self.cos, self.sin)

    def tables(self, want):
        return dominus_ultra_paged_tables(self.table, self.lens, want, self.ring, self.state, BLOCK, 1)

    def attend(self, q, lens):
        return dominus_ultra_decode_paged(q, self.k8, self.v8, self.ks, self.vs, self.table, lens, self.cos, self.sin)

    def step(self, q, k, v, want):
        slots, lens, _ = self.tables(want)
        self.write(k, v, slots, self.lens)
        return self.attend(q, lens)


def _expected(seed=1):
    s = _Step(seed)
    return s.step(s.q, s.k, s.v, s.lens + 1)


def _slow():
    """Some milliseconds of work on the current stream."""
    x = torch.ones(4096, 4096, device=DEV)
    for _ in range(8):
        x = x @ x * 1e-4
    return x


def _late(t):
    """The tensor's values, written by the current stream after some milliseconds of other work."""
    buf = torch.zeros_like(t)
    torch.cuda.synchronize()
    _slow()
    buf.copy_(t)
    return buf


@pytest.mark.parametrize("late", ["q", "k", "v", "want"])
def test_an_input_from_another_stream(late):
    want = _expected()
    s = _Step(1)
    args = dict(q=s.q, k=s.k, v=s.v, want=s.lens + 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        args[late] = _late(args[late])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(s.step(**args), want)


@pytest.mark.parametrize("late", ["q", "k", "v", "want"])
def test_an_input_copied_from_the_host(late):
    want = _expected()
    s = _Step(1)
    args = dict(q=s.q, k=s.k, v=s.v, want=s.lens + 1)
    host = args[late].cpu().pin_memory()
    args[late] = torch.zeros_like(args[late])
    torch.cuda.synchronize()
    _slow()
    args[late].copy_(host, non_blocking=True)
    assert torch.equal(s.step(**args), want)


def test_each_call_on_a_stream_of_its_own():
    want = _expected()
    s = _Step(1)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        _slow()
        slots, lens, _ = s.tables(s.lens + 1)
    streams[1].wait_stream(streams[0])
    with torch.cuda.stream(streams[1]):
        s.write(s.k, s.v, slots, s.lens)
        _slow()
    streams[2].wait_stream(streams[1])
    with torch.cuda.stream(streams[2]):
        out = s.attend(s.q, lens)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_a_capture_that_forks_and_joins():
    """Two steps in one graph: tables on the capture's stream, each step's write and attention on a fork."""
    want = [_expected(i) for i in (1, 2)]
    steps = [_Step(i) for i in (1, 2)]
    saved = [(s.k8.view(torch.uint8).clone(), s.v8.view(torch.uint8).clone(), s.ks.clone(), s.vs.clone(), s.table.clone()) for s in steps]
    q = [torch.zeros_like(s.q) for s in steps]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in steps:
        s.attend(s.q, s.lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        made = [s.tables(s.lens + 1) for s in steps]
        outs = []
        for i, s in enumerate(steps):
            side[i].wait_stream(main)
            with torch.cuda.stream(side[i]):
                s.write(s.k, s.v, made[i][0], s.lens)
        for i, s in enumerate(steps):  # each attention waits for both writes
            side[i].wait_stream(side[1 - i])
            with torch.cuda.stream(side[i]):
                outs.append(s.attend(q[i], made[i][1]))
        for x in side:
            main.wait_stream(x)
        outs = [o.clone() for o in outs]
    for _ in range(3):
        for s, (k, v, ks, vs, t) in zip(steps, saved):
            s.k8.view(torch.uint8).copy_(k)
            s.v8.view(torch.uint8).copy_(v)
            s.ks.copy_(ks)
            s.vs.copy_(vs)
            s.table.copy_(t)
        for dst, s in zip(q, steps):
            dst.copy_(s.q)
        graph.replay()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
            o.zero_()


@pytest.mark.parametrize("heads,kv_heads,dim,block", [(16, 8, 64, 128), (32, 8, 128, 16), (8, 8, 256, 64)])
def test_steps_back_to_back_equal_steps_apart(heads, kv_heads, dim, block):
    """Steps whose scales grow nearly every time, launched without a pause and with the GPU idle between any
    two calls: each kernel sees what the one before it wrote, neighbours' scales in one line among it."""
    batch, steps, width = 48, 60, 128 // block + 2
    g = torch.Generator(device=DEV).manual_seed(4)
    cos, sin = precompute_rope_cos_sin(width * block, dim, DEV, torch.bfloat16)
    grow = [2.0 ** (i * 0.6) for i in range(steps)]
    q = [torch.randn(batch, heads, 1, dim, generator=g, device=DEV).bfloat16() for _ in range(steps)]
    kv = [[(torch.randn(batch, kv_heads, 1, dim, generator=g, device=DEV) * x).bfloat16() for _ in range(2)] for x in grow]
    first = torch.randint(1, block, (batch,), generator=g, device=DEV, dtype=torch.int32)

    def run(pause):
        n = batch * width
        k8, v8 = (torch.zeros(n, kv_heads, block, dim, device=DEV).to(torch.float8_e4m3fn) for _ in range(2))
        ks, vs = torch.zeros(n, kv_heads, device=DEV), torch.zeros(n, kv_heads, device=DEV)
        table, ring, state = torch.full((batch, width), -1, **I32), torch.arange(n, **I32), torch.tensor([0, n], **I32)
        lens, outs = torch.zeros(batch, **I32), []
        for i in range(steps):
            # (the first step brings a prompt of zeros, so that requests end in different rows)
            new = first if i == 0 else lens + 1
            k, v = kv[i] if i else (torch.zeros(batch, kv_heads, block, dim, device=DEV).bfloat16() for _ in range(2))
            slots, grown, state = dominus_ultra_paged_tables(table, lens, new, ring, state, block, k.shape[2])
            pause()
            dominus_ultra_paged_write(k, v, k8, v8, ks, vs, slots, lens, cos, sin)
            pause()
            lens = grown
            outs.append(dominus_ultra_decode_paged(q[i], k8, v8, ks, vs, table, lens, cos, sin))
            pause()
        return outs, (k8.view(torch.uint8), v8.view(torch.uint8), ks, vs, table, lens)

    apart, state_apart = run(torch.cuda.synchronize)
    for _ in range(3):
        together, state_together = run(lambda: None)
        assert all(torch.equal(a, b) for a, b in zip(together, apart))
        assert all(torch.equal(a, b) for a, b in zip(state_together, state_apart))
