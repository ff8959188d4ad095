"""Paged attention where a CTA runs through many chunks, against 64 bits: both ways of cutting a batch
over the CTAs, references that move, sinks, value scales far apart, and results with a piece missing, which
have to be told."""

from __future__ import annotations

import math

import pytest
import torch

from dominusultra_b200 import _lib, dominus_ultra_decode_paged, dominus_ultra_paged_write
from tests import _paged_exact as exact
from tests._paged_batches import EQUAL_RANGES, PIECES

pytestmark = pytest.mark.gpu

DEV = "cuda"
CASES = {**EQUAL_RANGES, **PIECES}


@pytest.fixture(autouse=True)
def _clean_status(cuda_device):
    _lib.read_status(reset=True)
    yield
    assert _lib.read_status(reset=True)[0] == 0, "a test left a device status"


def _batch(Hq, Hkv, D, block, lens, dtype, seed, rise=None):
    """Random keys and values; the values of the request's chunk c have 8 more in column c mod D, so that
    each chunk shows in the output. `rise`: the scores' spread instead, (from, to) along a request."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    width = max(1, -(-max(lens) // block))
    N = sum(-(-n // block) for n in lens) + 2
    perm = torch.randperm(N, generator=g, device=DEV).int()
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV)
    k = torch.randn(N, Hkv, block, D, generator=g, device=DEV)
    v = torch.randn(N, Hkv, block, D, generator=g, device=DEV) / 2
    q = torch.randn(len(lens), Hq, 1, D, generator=g, device=DEV)
    positions = max(1, max(lens))
    if rise is None:
        angle = torch.arange(positions, device=DEV).double()[:, None] / 10000.0 ** (torch.arange(0, D, 2, device=DEV) / D)
        cos, sin = angle.cos().to(dtype), angle.sin().to(dtype)
        q = q / 2
    else:
        cos, sin = torch.ones(positions, D // 2, device=DEV).to(dtype), torch.zeros(positions, D // 2, device=DEV).to(dtype)
        q = torch.zeros_like(q)
        q[..., 0] = math.sqrt(D)
        k = k / 8
    at = 0
    for b, n in enumerate(lens):
        m = -(-n // block)
        ids = perm[at : at + m]
        table[b, :m] = ids
        at += m
        page = torch.arange(m, device=DEV)
        v[ids.long(), :, :, page * block // 128 % D] += 8
        if rise is not None:
            x = torch.linspace(*rise, m * block, device=DEV).reshape(m, 1, block)
            k[ids.long(), :, :, 0] = x.expand(m, Hkv, block)
    (k8, ks), (v8, vs) = exact.encode(k), exact.encode(v)
    return q.to(dtype), k8, v8, ks, vs, table, lens, cos, sin


def _call(q, k, v, ks, vs, table, lens, cos, sin):
    return dominus_ultra_decode_paged(q, k, v, ks, vs, table, torch.tensor(lens, dtype=torch.int32, device=DEV), cos, sin)


def _within(got, want, bound):
    return (got.double() - want).abs() <= exact.tolerance(want, bound, got.dtype)


def _check(batch, told=True):
    got = _call(*batch)
    want, bound = exact.attend(*batch)
    ok = _within(got, want, bound)
    assert bool(ok.all()), f"worst {((got.double() - want).abs() / exact.tolerance(want, bound, got.dtype)).max():.3f} of the tolerance"
    if not told:
        return
    # The tolerance tells a wrong result: zeros, or one chunk of the longest request left out.
    q, k, v, ks, vs, table, lens, cos, sin = batch
    b = max(range(len(lens)), key=lambda i: lens[i])
    one = (q[b : b + 1], k, v, ks, vs, table[b : b + 1], [lens[b]], cos, sin)
    zero = ~_within(torch.zeros_like(want[b]).to(got.dtype), want[b], bound[b])
    assert bool(zero.any(-1).all())
    chunks = -(-lens[b] // 128)
    for c in {0, 1, chunks // 2, chunks - 2}:
        less, _ = exact.attend(*one, skip=(128 * c, 128 * c + 128))
        assert not bool(_within(less.to(got.dtype), want[b : b + 1], bound[b : b + 1]).all(-1).any()), c


@pytest.mark.parametrize("name", CASES)
def test_long(name):
    Hq, Hkv, D, block, lens, dtype = CASES[name]
    _check(_batch(Hq, Hkv, D, block, lens, dtype, len(lens) + D))


@pytest.mark.parametrize("rise", [(-40.0, 40.0), (40.0, -40.0), (-3.0, 3.0)])
@pytest.mark.parametrize("name", [
    "64 requests, 32 heads on 8 of 128", "40 requests, 64 heads on 8 of 128", "50 requests, 8 heads of 64",
    "45 requests, 16 heads on 8 of 64", "100 requests, 16 heads on one of 256", "200 requests, 6 heads on 2 of 16",
])
def test_long_with_moving_references(name, rise):
    """Scores that rise (or fall) by 80 or 6 over a request: the weights' reference moves in most chunks
    (or in none after the first)."""
    Hq, Hkv, D, block, lens, dtype = CASES[name]
    _check(_batch(Hq, Hkv, D, block, lens, dtype, 3, rise), told=False)


@pytest.mark.parametrize("drop", [14.0, 18.5, 22.6, 25.0])
@pytest.mark.parametrize("D,G", [(64, 1), (64, 2), (128, 4), (128, 8), (256, 1), (256, 8), (32, 8), (16, 3)])
def test_long_tail_behind_a_sink(D, G, drop):
    """The first key takes nearly all of the weight and has values of zero; 3999 keys 2^-drop of it each make
    the output. Requests enough that a CTA has all of a unit."""
    B, block, n = 600, 16, 4000
    pages = n // block
    q = torch.zeros(B, G, 1, D, dtype=torch.float16, device=DEV)
    q[..., 0] = 8.0
    k = torch.zeros(pages, 1, block, D, device=DEV)
    k[0, 0, 0, 0] = 1.0
    v = torch.rand(pages, 1, block, D, generator=torch.Generator(device=DEV).manual_seed(D), device=DEV) + 0.5
    v[0, 0, 0] = 0
    v8, vs = exact.encode(v)
    ks = torch.full((pages, 1), drop * math.log(2) * math.sqrt(D) / 8, device=DEV)
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None].repeat(B, 1)
    cos, sin = torch.ones(n, D // 2, device=DEV).half(), torch.zeros(n, D // 2, device=DEV).half()
    got = _call(q, k.to(exact.E4M3), v8, ks, vs, table, [n] * B, cos, sin)
    want, bound = exact.attend(q[:1], k.to(exact.E4M3), v8, ks, vs, table[:1], [n], cos, sin)
    assert bool((bound <= 0.03 * want).all())
    assert bool(_within(got, want, bound).all()), f"off by {((got.double() - want).abs() / want).max():.4f}"


def _scaled(Hq, Hkv, D, lens, dtype, seed, scales):
    """Values whose blocks of 16 have the scales `scales(block of the request)`, magnitudes within the scale."""
    block = 16
    g = torch.Generator(device=DEV).manual_seed(seed)
    width = max(lens) // block + 1
    N = len(lens) * width
    table = torch.randperm(N, generator=g, device=DEV).int().reshape(len(lens), width)
    k8, ks = exact.encode(torch.randn(N, Hkv, block, D, generator=g, device=DEV))
    v8 = (torch.rand(N, Hkv, block, D, generator=g, device=DEV) + 0.5).to(exact.E4M3)
    vs = torch.empty(N, Hkv, device=DEV)
    for i in range(width):
        vs[table[:, i].long()] = scales(i)
    q = torch.randn(len(lens), Hq, 1, D, generator=g, device=DEV).to(dtype)
    cos, sin = torch.ones(max(lens), D // 2, device=DEV).to(dtype), torch.zeros(max(lens), D // 2, device=DEV).to(dtype)
    return q, k8, v8, ks, vs, table, lens, cos, sin


@pytest.mark.parametrize("Hq,Hkv,D,lens", [
    (4, 1, 64, [32]), (8, 1, 128, [32, 300]), (2, 2, 256, [700]), (8, 2, 32, [3000]), (4, 1, 128, [2500] * 400), (1, 1, 16, [900] * 700),
])
@pytest.mark.parametrize("name,scales", [
    ("zeros first", lambda i: 2.0**-64 if i == 0 else 2.0**67),
    ("zeros last", lambda i: 2.0**119 if i == 0 else 2.0**-64),
    ("alternating", lambda i: 2.0**-64 if i % 2 else 2.0**119),
    ("largest", lambda i: 2.0**126 * 1.25),
    ("largest among others", lambda i: (2.0**126, 2.0**-64, 2.0**-10, 2.0**40)[i % 4]),
    ("rising by chunks", lambda i: 2.0 ** min(119, -64 + 10 * (i // 8))),
])
def test_value_scales_far_apart(Hq, Hkv, D, lens, name, scales):
    """The softmax's sum has every key's weight, whatever the scales of the values."""
    batch = _scaled(Hq, Hkv, D, lens, torch.bfloat16, D, scales)
    q, k, v, ks, vs, table, _, cos, sin = batch
    got = _call(*batch)
    m = min(len(lens), 3)
    want, bound = exact.attend(q[:m], k, v, ks, vs, table[:m], lens[:m], cos, sin)
    assert bool((bound <= 0.02 * want).all())
    assert bool(_within(got[:m], want, bound).all()), f"off by {((got[:m].double() - want).abs() / want).max():.4f}"


def test_a_block_of_zeros_beside_huge_values_from_the_writer():
    """A block whose values are all zero has the writer's smallest scale; its keys keep their weight."""
    D, block = 64, 16
    k = torch.zeros(1, 1, 32, D, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    v[:, :, 16:] = 2.0**80
    k8, v8 = (torch.zeros(2, 1, block, D, device=DEV).to(exact.E4M3) for _ in range(2))
    ks, vs = torch.zeros(2, 1, device=DEV), torch.zeros(2, 1, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    cos, sin = torch.ones(32, D // 2, device=DEV).bfloat16(), torch.zeros(32, D // 2, device=DEV).bfloat16()
    dominus_ultra_paged_write(k, v, k8, v8, ks, vs, torch.arange(32, **i32)[None], torch.zeros(1, **i32), cos, sin)
    assert vs.flatten().tolist() == [2.0**-64, 2.0**72]
    q = torch.randn(1, 2, 1, D, device=DEV).bfloat16()
    got = _call(q, k8, v8, ks, vs, torch.arange(2, **i32)[None], [32], cos, sin)
    assert bool((got == 2.0**79).all())


@pytest.mark.parametrize("name", ["64 requests, 32 heads on 8 of 128", "36 uneven requests, 32 heads on 8 of 64", "one of 70000, 2 heads on one of 16"])
def test_long_replayed_and_on_two_streams(name):
    """A captured call replayed, and eager calls on two streams beside it, give the eager call's bits."""
    Hq, Hkv, D, block, lens, dtype = CASES[name]
    q, k, v, ks, vs, table, lens, cos, sin = _batch(Hq, Hkv, D, block, lens, dtype, 9)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    call = lambda: dominus_ultra_decode_paged(q, k, v, ks, vs, table, n, cos, sin)  # noqa: E731
    want = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        out.zero_()
        graph.replay()
        for s in streams:
            with torch.cuda.stream(s):
                got.append(call())
        assert torch.equal(out, want)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in got)
