"""Requests whose own length is out of range, in calls whose requests share blocks (GPU): nobody knows which of such a
row's entries are its blocks, so none of them may go to another request."""

from __future__ import annotations

import pytest
import torch

from dominusultra_b200 import _lib, dominus_ultra_paged_compact, dominus_ultra_paged_fork
from tests import _paged_shared as plain
from tests.test_paged_blocks_gpu import _batch, _gen, _ints

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_status(cuda_device):
    _lib.read_status(reset=True)
    yield
    assert _lib.read_status(reset=True)[0] == 0, "a test left a device status"


def _fork(table, lens, sources, wanted, ring, state, block):
    r = _ints(ring)
    got = dominus_ultra_paged_fork(_ints(table), _ints(lens), _ints(sources), _ints(wanted), r, _ints(state), block)
    return [x.tolist() for x in got] + [r.tolist()]


@pytest.mark.parametrize("n", [33, -1, 2**31 - 1, -(2**31)])
def test_a_fork_gives_no_block_of_such_a_row_back(n):
    ring = [2, 3, -1, -1, -1]
    table, copies, lens, state, left = _fork([[0, 1], [0, 1]], [n, 20], [0, 1], [0, 0], ring, [0, 2], 16)
    assert _lib.read_status(reset=True)[:2] == [6, 0]
    assert table == [[0, 1], [-1, -1]] and copies == [[-1, -1]] * 2 and lens == [n, 0]
    assert state == [0, 2] and left == ring


def test_a_fork_lets_nobody_write_a_block_of_such_a_row():
    table, copies, lens, state, left = _fork([[0, 1], [0, 1]], [-5, 20], [0, 1], [7, 7], [2, 3, -1, -1], [0, 2], 16)
    assert _lib.read_status(reset=True)[:2] == [6, 0]
    assert table == [[0, 1], [2, -1]] and copies == [[-1, -1], [0, 2]] and lens == [-5, 7]
    assert state == [1, 1] and left == [2, 3, -1, -1]


def test_a_fork_reports_no_entry_of_such_a_row():
    table, *_ = _fork([[7, -1, 10**6], [0, 1, 2]], [-5, 48], [0, 1], [0, 48], [3, 4, 5, -1, -1, -1, -1, -1], [0, 3], 16)
    assert _lib.read_status(reset=True)[:2] == [6, 0]
    assert table == [[7, -1, 10**6], [0, 1, 2]]


@pytest.mark.parametrize("B,width,N", [(7, 5, 64), (64, 9, 700), (33, 200, 5000), (300, 4, 1500), (5, 2000, 20000)])
@pytest.mark.parametrize("seed", [0, 1])
def test_forks_beside_such_rows(B, width, N, seed):
    """Such a row is as one whose blocks are all of its entries, and which continues from nobody."""
    block, g = 16, _gen(seed + B)
    table, lens, free = _batch(B, width, block, N, seed)
    sources = torch.randint(0, B, (B,), generator=g).tolist()
    wanted = [int(torch.randint(0, lens[s] + 1, (1,), generator=g)) for s in sources]
    ring = free + [-1] * (N - len(free))
    lost = [b for b in range(B) if torch.rand(1, generator=g) < 0.3] or [0]
    bad, as_held, alone = list(lens), list(lens), list(sources)
    for b in lost:
        bad[b] = -1 - b if b % 2 else width * block + 1 + b
        as_held[b] = width * block
    for b, s in enumerate(sources):
        if b in lost or s in lost:
            alone[b] = -1
    got = _fork(table, bad, sources, wanted, ring, [0, len(free)], block)
    assert _lib.read_status(reset=True)[0] == 6
    left = list(ring)
    want = plain.fork(table, as_held, alone, wanted, left, [0, len(free)], block)
    for b in lost:
        want[2][b] = bad[b]
    assert got == [*want, left]


def _compact(table, lens, ring, state, block):
    got = dominus_ultra_paged_compact(_ints(table), _ints(lens), _ints(ring), _ints(state), block)
    return [x.tolist() for x in got]


def _compacted(table, lens, ring, state, block):
    """plain.compact, where no block in a row with a length out of range moves."""
    width, N = len(table[0]), len(ring)
    ok = [0 <= n <= width * block for n in lens]
    held = [plain.pages(n, block) if o else 0 for n, o in zip(lens, ok)]
    free = {ring[(state[0] + i) % N] for i in range(state[1])}
    used = {x for r, h in zip(table, held) for x in r[:h]}
    assert len(free) == state[1] and not free & used
    used -= {x for r, o in zip(table, ok) if not o for x in r}
    low = set(sorted(used | free)[: len(used)])
    moves = list(zip(sorted(used - low), sorted(free & low)))
    place = dict(moves)
    rows = [[place.get(x, x) for x in r[:h]] + [-1] * (width - h) if o else list(r) for r, h, o in zip(table, held, ok)]
    left = sorted((used | free) - low)
    return rows, [list(m) for m in moves] + [[-1, -1]] * (N // 2 - len(moves)), left + [-1] * (N - len(left)), [0, state[1]]


@pytest.mark.parametrize("n", [49, -1, 2**31 - 1, -(2**31)])
def test_a_compaction_moves_no_block_of_such_a_row(n):
    # 6 and 7 are held by both rows, 5 by the second only
    table, copies, ring, state = _compact([[6, 7, -1], [6, 7, 5]], [n, 48], [0, 1, 2, -1, -1, -1, -1, -1], [0, 3], 16)
    assert _lib.read_status(reset=True)[:2] == [6, 0]
    assert table == [[6, 7, -1], [6, 7, 0]] and copies == [[5, 0]] + [[-1, -1]] * 3
    assert ring == [1, 2, 5, -1, -1, -1, -1, -1] and state == [0, 3]


def test_a_compaction_with_a_ring_that_holds_a_block_in_use_beside_such_a_row():
    args = ([[6, 7], [6, 5]], [-1, 20], [6, 1, 2, -1, -1, -1, -1, -1], [0, 3])
    table, copies, ring, state = _compact(*args, 16)
    assert _lib.read_status(reset=True)[0] in (6, 7)
    assert table == args[0] and copies == [[-1, -1]] * 4 and ring == args[2] and state == args[3]


@pytest.mark.parametrize("B,width,N", [(7, 5, 64), (64, 9, 700), (33, 200, 9000), (1030, 3, 5000), (5, 2000, 20000), (100, 300, 70001)])
@pytest.mark.parametrize("part", [0.3, 1.0])
def test_compactions_beside_such_rows(B, width, N, part):
    block, g = 16, _gen(B + N)
    table, lens, free = _batch(B, width, block, N, B + N)
    count = int(len(free) * part)
    ring = [-1] * N
    for i in range(count):
        ring[(N - 1 + i) % N] = free[i]
    bad = list(lens)
    for b in [b for b in range(B) if torch.rand(1, generator=g) < 0.3] or [B - 1]:
        bad[b] = -1 - b if b % 2 else width * block + 1 + b
    got = _compact(table, bad, ring, [N - 1, count], block)
    assert _lib.read_status(reset=True)[0] == 6
    assert got == [*_compacted(table, bad, ring, [N - 1, count], block)]
