"""Free ring of the paged block tables: entries that are not block ids."""

from __future__ import annotations

import pytest
import torch

from dominusultra_b200 import _lib, dominus_ultra_paged_tables

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("value", [-1, 6, 2**31 - 1, -(2**31)])
@pytest.mark.parametrize("page", [0, 1, 2])
def test_damaged_entry_is_reported_where_it_is_given_back(cuda_device, value, page):
    """Request 1 ends and gives back a row with a damaged entry: the status names it, and the entries
    around it and other requests are as ever."""
    _lib.read_status(reset=True)
    row = [4, 1, 3]
    row[page] = value
    table = torch.tensor([[0, -1, -1], row, [2, -1, -1]], **I32)
    ring, state = torch.tensor([5, -9, -9, -9, -9, -9], **I32), torch.tensor([0, 1], **I32)
    old, new = torch.tensor([16, 40, 5], **I32), torch.tensor([17, 0, 6], **I32)
    slots, lens, left = dominus_ultra_paged_tables(table, old, new, ring, state, 16, 1)
    assert _lib.read_status(reset=True)[:3] == [7, 1, value & 0xFFFFFFFF]
    assert slots.tolist() == [[80], [-1], [37]] and lens.tolist() == [17, 0, 6]
    assert ring.tolist() == [5, *row, -9, -9] and left.tolist() == [1, 3]
    # the next request that is given it has no slot in it, and is named
    table = torch.full((1, 3), -1, **I32)
    slots, lens, _ = dominus_ultra_paged_tables(table, torch.zeros(1, **I32), torch.tensor([48], **I32), ring, left, 16, 48)
    assert _lib.read_status(reset=True)[:3] == [7, 0, value & 0xFFFFFFFF]
    assert table.tolist() == [row] and lens.tolist() == [48]
    assert [x >= 0 for x in slots[0].tolist()] == [i // 16 != page for i in range(48)]


def test_sound_entries_are_not_reported(cuda_device):
    _lib.read_status(reset=True)
    table = torch.tensor([[0, 5], [4, 1]], **I32)
    ring, state = torch.full((6,), -9, **I32), torch.tensor([3, 0], **I32)
    dominus_ultra_paged_tables(table, torch.tensor([32, 17], **I32), torch.zeros(2, **I32), ring, state, 16, 1)
    assert _lib.read_status(reset=True)[0] == 0 and ring.tolist() == [1, -9, -9, 0, 5, 4]
