"""Paged attention where a CTA runs through many chunks, against 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from dominusultra_b200 import _lib, dominus_ultra_decode_paged
from tests import _paged_exact as exact

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(autouse=True)
def _clean_status(cuda_device):
    _lib.read_status(reset=True)
    yield
    assert _lib.read_status(reset=True)[0] == 0, "a test left a device status"


def _call(q, k, v, ks, vs, table, lens, cos, sin):
    return dominus_ultra_decode_paged(q, k, v, ks, vs, table, torch.tensor(lens, dtype=torch.int32, device=DEV), cos, sin)


def _within(got, want, bound):
    return (got.double() - want).abs() <= exact.tolerance(want, bound, got.dtype)


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
