"""The borders of the calls on shared paged caches: the largest sets, the row counts at which an extension lays its
rows out otherwise, maxima that move with every tile, scratch that holds anything, graphs side by side."""

from __future__ import annotations

import pytest
import torch

from dominusultra_b200 import _lib, dominus_ultra_extend_paged, dominus_ultra_paged_compact, dominus_ultra_paged_fork, paged
from tests import _paged_shared as plain
from tests.test_paged_blocks_gpu import _batch, _check_fork, _gen, _ints
from tests.test_paged_extend_gpu import BF, HF, _call, _case, _check

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_status(cuda_device):
    _lib.read_status(reset=True)
    yield
    assert _lib.read_status(reset=True)[0] == 0, "a test left a device status"


def _dirty():
    """NaN in whatever scratch the calls of this process keep."""
    torch.cuda.synchronize()
    for pair in paged._SCRATCH.values():
        pair[4].fill_(0xFF)
    torch.cuda.synchronize()


@pytest.mark.parametrize("B,width,N", [(8192, 2, 240000), (8192, 40, 200000), (1, 9, 524287), (1025, 129, 100000)])
def test_largest_forks(B, width, N):
    block = 16
    table, lens, free = _batch(B, width, block, N, 3)
    g = _gen(B)
    sources = torch.randint(0, B, (B,), generator=g).tolist()
    wanted = [int(torch.randint(0, lens[s] + 1, (1,), generator=g)) for s in sources]
    head = N - 5
    ring = [-1] * N
    for i, x in enumerate(free):
        ring[(head + i) % N] = x
    _check_fork(table, lens, sources, wanted, ring, [head, len(free)], block)


@pytest.mark.parametrize("B,width,N", [(8192, 3, 770000), (3, 4000, 770000), (700, 131, 262144)])
def test_largest_compactions(B, width, N):
    block = 16
    table, lens, free = _batch(B, width, block, N, 4)
    keep = [x for i, x in enumerate(free) if i % 3]  # (the others are somebody else's)
    head = N - 7
    ring = [-1] * N
    for i, x in enumerate(keep):
        ring[(head + i) % N] = x
    args = (_ints(table), _ints(lens), _ints(ring), _ints([head, len(keep)]))
    _dirty()
    got = dominus_ultra_paged_compact(*args, block)
    want = plain.compact(table, lens, ring, [head, len(keep)], block)
    for x, y in zip(got, want):
        assert x.tolist() == y


@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("rows", [1, 8, 9, 16, 17, 31, 32, 33, 48, 64, 65, 128, 129])
def test_rows_of_an_item(D, rows):
    # (one head per key head: as many rows as tokens; the second request has one token)
    c = _case(2, 2, D, rows, [700, 1000, 0], [rows, 1, rows], 16, BF, seed=rows + D)
    _call(c)
    _dirty()
    _check(c)


@pytest.mark.parametrize("D,T", [(64, 3), (128, 40), (128, 100), (128, 200), (256, 30), (64, 300)])
def test_a_maximum_that_moves_with_every_tile(D, T):
    c = _case(2, 2, D, T, [2000], [T], 16, HF, seed=D + T, spread=0)
    row = c["table"][0].long()
    row = row[row >= 0]
    c["ks"][row] *= torch.linspace(0.05, 4.0, len(row), device="cuda")[:, None]
    _check(c)


@pytest.mark.parametrize("T", [1, 40, 70, 200])
@pytest.mark.parametrize("width", [1, 3, 4, 5, 8, 9])
def test_tables_of_few_tiles(T, width):
    # 16 to 144 positions: one key tile, or just more
    n = 16 * width
    new = min(T, n)
    _check(_case(4, 2, 128, T, [n - new, 0], [new, new], 16, BF, seed=T + width, width=width))


def test_compactions_in_two_graphs_at_once():
    block, N, B, width = 16, 3000, 40, 30
    cases = []
    for seed in (1, 2):
        table, lens, free = _batch(B, width, block, N, seed)
        ring = free + [-1] * (N - len(free))
        args = [_ints(x) for x in (table, lens, ring, [0, len(free)])]
        want = plain.compact(table, lens, ring, [0, len(free)], block)
        dominus_ultra_paged_compact(*args, block)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = dominus_ultra_paged_compact(*args, block)
        cases.append((g, got, want, torch.cuda.Stream(), args))  # (the graph reads its inputs where they are)
    torch.cuda.synchronize()
    for _ in range(5):
        for g, got, _, s, _ in cases:
            with torch.cuda.stream(s):
                for x in got:
                    x.fill_(-7)
                g.replay()
    torch.cuda.synchronize()
    for _, got, want, _, _ in cases:
        for x, y in zip(got, want):
            assert x.tolist() == y


def test_extensions_and_compactions_share_a_streams_scratch():
    c = _case(8, 2, 64, 4, [3000, 20], [4, 4], 16, BF, seed=1)
    table, lens, free = _batch(20, 30, 16, 2000, 5)
    ring = free + [-1] * (2000 - len(free))
    args = [_ints(x) for x in (table, lens, ring, [0, len(free)])]
    want, sets = _call(c), plain.compact(table, lens, ring, [0, len(free)], 16)
    for _ in range(5):
        out = _call(c)
        got = dominus_ultra_paged_compact(*args, 16)
        again = dominus_ultra_extend_paged(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], _ints(c["past"]), _ints(c["lens"]), c["cos"], c["sin"])
        assert torch.equal(out, want) and torch.equal(again, want)
        assert all(x.tolist() == y for x, y in zip(got, sets))


def test_forks_on_two_streams_at_once():
    block, N, B, width = 16, 4000, 64, 30
    cases = []
    for seed in (1, 2):
        table, lens, free = _batch(B, width, block, N, seed)
        g = _gen(seed)
        sources = torch.randint(0, B, (B,), generator=g).tolist()
        wanted = [lens[s] for s in sources]
        ring = free + [-1] * (N - len(free))
        args = [_ints(x) for x in (table, lens, sources, wanted, ring, [0, len(free)])]
        want = plain.fork(table, lens, sources, wanted, list(ring), [0, len(free)], block)
        cases.append((args, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (args, _, s) in enumerate(cases):
            with torch.cuda.stream(s):
                got[i].append(dominus_ultra_paged_fork(*args, block))
    torch.cuda.synchronize()
    for outs, (_, want, _) in zip(got, cases):
        for out in outs:
            assert all(x.tolist() == y for x, y in zip(out, want))
