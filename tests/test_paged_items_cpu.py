"""Items of the paged extension that lie in one CTA with others behind them (no GPU): that the batches of
test_paged_items_gpu.py reach them, and that warps keep to their own bytes between two of them."""

from __future__ import annotations

import re

import pytest

from dominusultra_b200 import build
from tests import _paged_items as items
from tests._paged_items import UNCUT


def _followed(case):
    """Rows of the items that lie in one CTA with another fragment behind them."""
    Hq, Hkv, D, T, new, past, _ = case
    return [f[3] for cta in items.split(past, new, Hq, Hkv, D, T) for f in cta[:-1] if f[6] == 1]


@pytest.mark.parametrize("name", UNCUT)
def test_every_tile_is_in_one_fragment(name):
    Hq, Hkv, D, T, new, past, _ = UNCUT[name]
    _, _, keys, _ = items.plan(T, Hq // Hkv, D)
    seen = {}
    for cta in items.split(past, new, Hq, Hkv, D, T):
        for b, h, i, rows, lo, hi, count in cta:
            seen.setdefault((b, h, i), []).append((lo, hi, rows, count))
    assert sum(x[0][2] for x in seen.values()) == sum(new) * Hq
    for (b, _, i), parts in seen.items():
        assert parts[0][0] == 0 and all(x[1] == y[0] for x, y in zip(parts, parts[1:]))
        assert all(x[3] == len(parts) for x in parts) and (parts[-1][1] - 1) * keys < past[b] + new[b]


@pytest.mark.parametrize("name", UNCUT)
def test_whole_items_have_others_behind_them(name):
    assert len(_followed(UNCUT[name])) >= 100


@pytest.mark.parametrize("D", [128, 256])
def test_last_row_tiles_leave_one_two_and_three_warps_empty(D):
    rows = {r for case in UNCUT.values() if case[2] == D for r in _followed(case)}
    assert {-(-(r % 128) // 32) for r in rows} >= {1, 2, 3}


@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
def test_offsets_are_a_permutation_and_meet_no_bank_twice(D):
    pieces = 2 * D // 16
    at = [items.offset(r, c, D) for r in range(128) for c in range(pieces)]
    assert sorted(at) == list(range(0, 128 * 2 * D, 16))
    for c in range(pieces):  # a row per lane, eight lanes at a time
        for r in range(0, 128, 8):
            assert len({items.offset(r + i, c, D) // 16 % 8 for i in range(8)}) == 8
    for first in range(0, 128 * pieces, 8):  # neighbouring lanes with neighbouring pieces
        assert len({items.offset(x // pieces, x % pieces, D) // 16 % 8 for x in range(first, first + 8)}) == 8


@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
def test_rows_one_after_the_other_would_be_other_warps_bytes(D):
    """What the outputs' place among the query rows is for."""
    for warp in range(4):
        rows = range(32 * warp, 32 * warp + 32)
        queries = {items.offset(r, c, D) for r in rows for c in range(2 * D // 16)}
        in_turn = {r * 2 * D + 16 * c for r in rows for c in range(2 * D // 16)}
        assert (queries == in_turn) == (D <= 64)


def test_the_kernel_addresses_the_row_tile_by_that_offset_only():
    """Query rows and outputs are in the same bytes of the same warp, and between two items nothing else orders the
    warps of a stream whose rows have one part."""
    text = re.sub(r"//[^\n]*", "", (build.CSRC / "extend_paged_sm100.cuh").read_text())
    uses = re.findall(r"\bq_tile\b(?! =)\s*(\+?\s*\w*(?:<SPAN>\(128,)?)", text)
    assert len(uses) >= 6
    assert all(re.fullmatch(r"\+ swz_chunk_offset<SPAN>\(128,", u) for u in uses), uses
