"""How the paged attention cuts batches over its CTAs (no GPU)."""

from __future__ import annotations

import pytest

from tests import _paged_exact as exact
from tests._paged_batches import EQUAL_RANGES, PIECES


def _split(case):
    Hq, Hkv, D, block, lens, _ = case
    width = max(1, -(-max(lens) // block))
    return exact.split(lens, Hq, Hkv, D, block, width)


def _whole(case, ctas):
    """Every chunk of every unit is in exactly one fragment, and fragments know how many there are."""
    Hq, Hkv, D, _, lens, _ = case
    ups = exact.shape(Hq, Hkv, D)[1]
    seen = {}
    for frags in ctas:
        for unit, a, b, nf in frags:
            seen.setdefault(unit, []).append((a, b, nf))
    assert len(seen) == len(lens) * ups
    for unit, parts in seen.items():
        parts.sort()
        assert parts[0][0] == 0 and parts[-1][1] == max(1, -(-lens[unit // ups] // 128))
        assert all(x[1] == y[0] for x, y in zip(parts, parts[1:]))
        assert all(x[2] == len(parts) for x in parts)


@pytest.mark.parametrize("name", EQUAL_RANGES)
def test_equal_ranges(name):
    case = EQUAL_RANGES[name]
    ctas, pieces = _split(case)
    assert not pieces
    _whole(case, ctas)
    assert max(b - a for f in ctas for _, a, b, _ in f) >= 9  # beyond the stages of K and V (at most 8)
    assert any(nf >= 2 for f in ctas for *_, nf in f)
    assert any(len(f) >= 2 for f in ctas)


def test_equal_ranges_reach_every_way_of_joining():
    many = both = False
    for case in EQUAL_RANGES.values():
        ctas, _ = _split(case)
        many |= any(nf >= 4 for f in ctas for *_, nf in f)
        both |= any(len(f) >= 2 and f[0][3] > 1 and f[-1][3] > 1 for f in ctas)  # two units to join at most
    assert many and both
    assert {exact.shape(q, k, d)[0] for q, k, d, *_ in EQUAL_RANGES.values()} == {1, 2, 4, 8}
    assert {c[2] for c in EQUAL_RANGES.values()} == {16, 32, 64, 128, 256}


@pytest.mark.parametrize("name", PIECES)
def test_pieces(name):
    case = PIECES[name]
    ctas, pieces = _split(case)
    assert pieces
    _whole(case, ctas)
    assert max(len(f) for f in ctas) == 1


def test_pieces_reach_long_fragments_and_long_joins():
    sizes, joins = [], []
    for case in PIECES.values():
        ctas, _ = _split(case)
        sizes.append(max(b - a for f in ctas for _, a, b, _ in f))
        joins.append(max(nf for f in ctas for *_, nf in f))
    assert max(sizes) >= 16 and max(joins) > 128
