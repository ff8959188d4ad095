"""How the paged attention carries its weights (no GPU)."""

from __future__ import annotations

import torch

from tests import _paged_exact as exact


def test_four_parts_are_the_fp16_weight():
    """Every fp16 weight in [0, 256], the smallest ones too, is the sum of its four parts."""
    w = torch.arange(0, 0x5C00 + 1, dtype=torch.int16).view(torch.float16).double()
    assert w[-1] == 256.0
    parts, total = exact.parts_of_weight(w)
    assert len(parts) == 4 and torch.equal(total, w)
    assert all(p.abs().max() <= 256 for p in parts)


def test_three_parts_close_together_lose_small_weights():
    """Why the parts are four: three with 2^4 between them end at 2^-18, which carries a weight of 2^-17.9
    as twice itself and one below 2^-18 as nothing."""
    _, total = exact.parts_of_weight(torch.tensor([2.0**-17.9, 2.0**-18.1], dtype=torch.float64), (4, 4))
    assert total[0] > 1.8 * 2.0**-17.9 and total[1] == 0


def test_three_parts_five_apart_are_the_larger_weights():
    w = torch.arange(0, 0x5C00 + 1, dtype=torch.int16).view(torch.float16).double()
    _, total = exact.parts_of_weight(w, (5, 5))
    assert torch.equal(total[w >= 2.0**-9], w[w >= 2.0**-9]) and not torch.equal(total, w)


def test_the_scaled_sum_stays_in_range():
    """The softmax's sum is kept 2^24 times too large: 2^27 of the largest terms fit, and the smallest that
    the largest of a warp can be is a normal number with 28 octaves below it."""
    largest = 2.0 ** (8 + 64 + 24)  # a weight of 2^8 over the smallest value scale
    smallest = 2.0 ** (7 - 128 + 24)  # the reference's own key over the largest value scale
    assert largest * 2**27 < torch.finfo(torch.float32).max
    assert smallest * 2.0**-28 >= torch.finfo(torch.float32).tiny
