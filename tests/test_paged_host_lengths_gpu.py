"""Lengths of the paged extension of which only one is on the CPU (GPU)."""

from __future__ import annotations

import pytest
import torch

from dominusultra_b200 import _lib, dominus_ultra_extend_paged
from tests.test_paged_extend_gpu import BF, _call, _case, _ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [-1, 129, 2**31 + 5])
def test_lengths_before_the_new_tokens_are_checked_on_the_cpu(cuda_device, bad):
    c = _case(4, 2, 64, 4, [50, 60], [4, 4], 16, BF, seed=8, width=8)
    args = [c[x] for x in ("q", "k", "v", "ks", "vs", "table")]
    good = dominus_ultra_extend_paged(*args, torch.tensor(c["past"]), _ints(c["lens"]), c["cos"], c["sin"])
    assert torch.equal(good, _call(c))
    _lib.read_status(reset=True)
    with pytest.raises(ValueError, match=r"past_seqlens\[1\]"):
        dominus_ultra_extend_paged(*args, torch.tensor([50, bad]), _ints(c["lens"]), c["cos"], c["sin"])
    assert _lib.read_status(reset=True)[0] == 0
