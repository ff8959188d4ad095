"""Pairs of a copy whose ids are both below the range: {-1, -1} is no copy, all others are reported (GPU)."""

from __future__ import annotations

import pytest
import torch

from dominusultra_b200 import _lib, dominus_ultra_paged_copy

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pair", [[-1, -1], [-2, -2], [-1, -2], [-2, -1], [-(2**31), -1], [-7, -(2**31)]])
def test_pairs_below_the_range(cuda_device, pair):
    _lib.read_status(reset=True)
    k = torch.arange(4 * 256, device="cuda").to(torch.uint8).reshape(4, 1, 16, 16)
    v, s = k + 1, torch.arange(4.0, device="cuda").reshape(4, 1)
    w = s + 4
    want = [x.clone() for x in (k, v, s, w)]
    for x in want:
        x[2] = x[3]
    copies = torch.tensor([[3, 2], pair], dtype=torch.int32, device="cuda")
    dominus_ultra_paged_copy(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), s, w, copies)
    assert all(torch.equal(x, y) for x, y in zip((k, v, s, w), want))
    assert _lib.read_status(reset=True)[:2] == ([0, 0] if pair == [-1, -1] else [7, 1])
