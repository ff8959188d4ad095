"""Forks, copies and compactions of the paged cache's blocks on the GPU against the plain integers of
tests/_paged_shared.py."""

from __future__ import annotations

import pytest
import torch

from dominusultra_b200 import _lib, dominus_ultra_paged_compact, dominus_ultra_paged_copy, dominus_ultra_paged_fork
from tests import _paged_shared as plain

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _status():
    return _lib.read_status(reset=True)


@pytest.fixture(autouse=True)
def _clean_status(cuda_device):
    _status()
    yield
    assert _status()[0] == 0, "a test left a device status"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def _check_fork(table, lens, sources, wanted, ring, state, block, stream=None):
    t, r, s = _ints(table), _ints(ring), _ints(state)
    got = dominus_ultra_paged_fork(t, _ints(lens), _ints(sources), _ints(wanted), r, s, block)
    again = dominus_ultra_paged_fork(t, _ints(lens), _ints(sources), _ints(wanted), r, s, block)  # the same inputs, the same values
    ring = list(ring)
    want = plain.fork(table, lens, sources, wanted, ring, state, block)
    for x, y, z in zip(got, want, again):
        assert x.tolist() == y
        assert z.tolist() == y
    assert r.tolist() == ring and t.tolist() == table and s.tolist() == list(state)
    return want


def _batch(B, width, block, N, seed, shared=True):
    """A table whose rows share beginnings of whole blocks with rows before them, and a ring of the rest."""
    g = _gen(seed)
    order = torch.randperm(N, generator=g).tolist()
    table, lens = [], []
    for b in range(B):
        n = int(torch.randint(0, width * block + 1, (1,), generator=g))
        need, row = plain.pages(n, block), []
        if shared and b and int(torch.randint(0, 2, (1,), generator=g)):
            s = int(torch.randint(0, b, (1,), generator=g))
            row = table[s][: int(torch.randint(0, min(lens[s], n) // block + 1, (1,), generator=g))]
        take = min(need - len(row), len(order))
        row = row + order[:take]
        order = order[take:]
        n = min(n, len(row) * block)
        table.append(row + [-1] * (width - len(row)))
        lens.append(n)
    return table, lens, order


@pytest.mark.parametrize("B,width,block,N", [(1, 1, 16, 1), (1, 1, 128, 33), (2, 3, 16, 40), (7, 5, 32, 64), (64, 9, 16, 700), (33, 200, 64, 5000), (300, 4, 128, 1500), (1030, 3, 16, 4000), (5, 2000, 16, 20000)])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_fork(B, width, block, N, seed):
    g = _gen(seed + 10 * B)
    table, lens, free = _batch(B, width, block, N, seed)
    sources = torch.where(torch.rand(B, generator=g) < 0.5, torch.arange(B), torch.randint(0, B, (B,), generator=g)).tolist()
    wanted = [int(torch.randint(0, lens[s] + 1, (1,), generator=g)) if int(torch.randint(0, 3, (1,), generator=g)) else lens[s] for s in sources]
    head = int(torch.randint(0, N, (1,), generator=g))
    count = len(free) if seed != 2 else min(len(free), B // 8)
    ring = [-1] * N
    for i in range(count):
        ring[(head + i) % N] = free[i]
    _check_fork(table, lens, sources, wanted, ring, [head, count], block)


def test_fork_rotates_beams_without_copies():
    # a permutation of the requests: each last block changes hands
    table, lens = [[3, 4], [5, 6], [7, 8]], [20, 20, 20]
    out = _check_fork(table, lens, [1, 2, 0], [20, 20, 20], list(range(9, 12)) + [-1] * 9, [0, 3], 16)
    assert out[0] == [[5, 6], [7, 8], [3, 4]] and out[1] == [[-1, -1]] * 3 and out[3] == [0, 3]


def test_fork_of_one_into_all():
    out = _check_fork([[3, 4], [5, 6], [7, 8]], [20, 20, 20], [1, 1, 1], [20, 20, 20], [0, 1, 2] + [-1] * 9, [0, 3], 16)
    # the lowest request keeps the partly filled block, the others get copies; what 0 and 2 held is free
    assert out[0] == [[5, 6], [5, 0], [5, 1]] and out[1] == [[-1, -1], [6, 0], [6, 1]] and out[3] == [2, 5]


def test_fork_into_a_block_that_another_holds_whole():
    # request 0 shrinks into a block that request 1 holds whole: it gets a copy, and the lowest rule does not apply
    out = _check_fork([[0, -1], [0, 1]], [16, 20], [0, 1], [5, 20], [2] + [-1] * 4, [0, 1], 16)
    assert out[0] == [[2, -1], [0, 1]] and out[1] == [[0, 2], [-1, -1]]


def test_fork_without_a_free_block_is_cut():
    out = _check_fork([[0, 1], [2, -1]], [20, 3], [0, 0], [20, 20], [-1] * 8, [0, 0], 16)
    assert out[2] == [20, 16] and out[0] == [[0, 1], [0, -1]] and out[3] == [0, 1]


def test_fork_ends_everything():
    out = _check_fork([[0, 1], [0, 2]], [20, 30], [0, 1], [0, 0], [-1] * 5, [4, 0], 16)
    assert out[3] == [4, 3]


def test_fork_many_requests_end_in_one_block():
    B = 777
    out = _check_fork([[0]] * B, [5] + [0] * (B - 1), [0] * B, [5] * B, list(range(1, B + 1)) + [-1], [0, B], 16)
    assert out[1][0] == [-1, -1] and out[1][-1] == [0, B - 1]


@pytest.mark.parametrize("what", ["source", "source_low", "wanted", "wanted_low", "len", "len_low", "len_of_source"])
def test_fork_out_of_range(what):
    table, lens, sources, wanted = [[0, 1], [2, 3], [4, 5]], [20, 25, 32], [1, 1, 2], [25, 20, 32]
    if what == "source":
        sources[0] = 3
    elif what == "source_low":
        sources[0] = -1
    elif what == "wanted":
        wanted[0] = 26
    elif what == "wanted_low":
        wanted[0] = -2
    elif what == "len":
        lens[0] = 33
    elif what == "len_low":
        lens[0] = -1
    else:
        lens[1] = 40
    _check_fork(table, lens, sources, wanted, list(range(6, 16)) + [-1] * 2, [0, 4], 16)
    assert _status()[0] == 6


@pytest.mark.parametrize("state", [[-1, 2], [12, 2], [0, 13], [0, -1], [0, 11]])
def test_fork_ring_state_out_of_range(state):
    # (the last: more given back than the ring has room for)
    _check_fork([[0, 1], [2, 3]], [20, 25], [0, 0], [20, 20], list(range(12)), state, 16)
    assert _status()[0] == 7


def test_fork_damaged_entries():
    _check_fork([[0, 99], [-7, 3]], [20, 25], [0, 0], [20, 3], list(range(4, 12)) + [-1] * 4, [0, 4], 16)
    assert _status()[0] == 7


def test_fork_damaged_ring():
    out = _check_fork([[0], [1]], [5, 5], [0, 0], [5, 5], [77, 2, 3, 4], [0, 3], 16)
    assert out[1][1] == [0, 77] and _status()[:3] == [7, 1, 77]


def test_fork_int64_and_host_lengths():
    t, r, s = _ints([[0, 1], [2, -1]]), _ints([3, 4, 5, -1, -1, -1]), _ints([0, 3])
    lens, src, want = (torch.tensor(x, dtype=torch.int64) for x in ([20, 7], [0, 0], [20, 20]))
    got = dominus_ultra_paged_fork(t, lens, src.to(DEV), want, r, s, 16)
    assert [x.tolist() for x in got] == [[[0, 1], [0, 3]], [[-1, -1], [1, 3]], [20, 20], [1, 3]]
    with pytest.raises(ValueError, match="sources"):
        dominus_ultra_paged_fork(t, lens, src + 5, want, r, s, 16)
    with pytest.raises(ValueError, match="cache_seqlens"):
        dominus_ultra_paged_fork(t, lens + 50, src, want, r, s, 16)


# ---------------------------------------------------------------------------------------- compact


def _check_compact(table, lens, ring, state, block):
    t, r, s = _ints(table), _ints(ring), _ints(state)
    got = dominus_ultra_paged_compact(t, _ints(lens), r, s, block)
    want = plain.compact(table, lens, ring, state, block)
    for x, y in zip(got, want):
        assert x.tolist() == y
    assert t.tolist() == table and r.tolist() == ring and s.tolist() == list(state)
    return want


@pytest.mark.parametrize("B,width,block,N", [(1, 1, 16, 1), (1, 1, 16, 2), (2, 3, 16, 40), (7, 5, 32, 64), (64, 9, 16, 700), (33, 200, 64, 9000), (1030, 3, 16, 5000), (5, 2000, 16, 20000), (100, 300, 16, 70001)])
@pytest.mark.parametrize("part", [0.0, 0.3, 1.0])
def test_compact(B, width, block, N, part):
    table, lens, free = _batch(B, width, block, N, B + N)
    count = int(len(free) * part)
    head = N - 1
    ring = [-1] * N
    for i in range(count):
        ring[(head + i) % N] = free[i]
    _check_compact(table, lens, ring, [head, count], block)


def test_compact_nothing_in_use_and_nothing_free():
    _check_compact([[-1, -1]], [0], [2, 0, 1], [1, 3], 16)
    _check_compact([[1, 2]], [32], [-1, -1, -1], [0, 0], 16)


def test_compact_leaves_others_blocks():
    # ids 0 and 3 are neither held nor free
    out = _check_compact([[5, 4]], [20], [1, 2, -1, -1, -1, -1], [0, 2], 16)
    assert out[0] == [[2, 1]] and out[1] == [[4, 1], [5, 2], [-1, -1]] and out[2][:2] == [4, 5]


@pytest.mark.parametrize("ring,state", [([1, 1, 2, 3], [0, 2]), ([1, 0, 2, 3], [0, 2]), ([9, 1, 2, 3], [0, 2]), ([1, 2, 3, 3], [4, 2]), ([1, 2, 3, 3], [0, 5]), ([1, 2, 3, 3], [0, -1])])
def test_compact_ring_out_of_range(ring, state):
    _check_compact([[0, -1]], [5], ring, state, 16)
    assert _status()[0] == 7


@pytest.mark.parametrize("n", [-1, 33])
def test_compact_length_out_of_range(n):
    _check_compact([[6, 7], [5, -1]], [n, 5], [0, 1, 2, 3, 4, 8, 9, -1, -1, -1], [0, 4], 16)
    assert _status()[0] == 6


def test_compact_damaged_entry_stays():
    _check_compact([[6, 77], [-3, 5]], [20, 20], [0, 1, 2, 3, 4, 8, 9, -1, -1, -1], [0, 4], 16)
    assert _status()[0] == 7


# ------------------------------------------------------------------------------------------- copy


@pytest.mark.parametrize("Hkv,block,D", [(1, 16, 16), (1, 16, 64), (3, 16, 16), (8, 16, 128), (2, 128, 256), (5, 32, 32), (40, 16, 64)])
@pytest.mark.parametrize("n", [1, 7, 300])
def test_copy(Hkv, block, D, n):
    g = _gen(n + D)
    N = 2 * n + 3
    caches = [torch.randint(0, 256, (N, Hkv, block, D), generator=g, dtype=torch.uint8).to(DEV) for _ in range(2)]
    scales = [torch.rand(N, Hkv, generator=g).to(DEV) for _ in range(2)]
    pairs = torch.randperm(N, generator=g)[: 2 * n].reshape(n, 2)
    pairs[1::3] = -1
    want = [x.clone() for x in caches + scales]
    for src, dst in pairs.tolist():
        if src >= 0:
            for x in want:
                x[dst] = x[src]
    dominus_ultra_paged_copy(*(x.view(torch.float8_e4m3fn) for x in caches), *scales, pairs.int().to(DEV))
    for x, y in zip(caches + scales, want):
        assert torch.equal(x, y)


def test_copy_of_nothing():
    k = torch.zeros(2, 1, 16, 16, device=DEV).to(torch.float8_e4m3fn)
    s = torch.ones(2, 1, device=DEV)
    dominus_ultra_paged_copy(k, k.clone(), s, s.clone(), torch.empty(0, 2, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("pair", [[0, 4], [4, 0], [-1, 1], [1, -1], [2**31 - 1, 0]])
def test_copy_out_of_range_is_left_out(pair):
    k = torch.arange(4 * 256, device=DEV).to(torch.uint8).reshape(4, 1, 16, 16)
    v, s = k + 1, torch.arange(4.0, device=DEV).reshape(4, 1)
    w = s + 4
    before = [x.clone() for x in (k, v, s, w)]
    dominus_ultra_paged_copy(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), s, w, _ints([pair, [3, 2]]))
    for x, y in zip((k, v, s, w), before):
        y[2] = y[3]
        assert torch.equal(x, y)
    assert _status()[:2] == [7, 0]


# -------------------------------------------------------------------------- streams and captures


def test_fork_copy_compact_captured_and_replayed():
    block, B, width, N, Hkv, D = 16, 6, 5, 64, 2, 64
    g = _gen(4)
    t, ln, ring, state = (_ints(x) for x in ([[-1] * width] * B, [0] * B, list(range(N)), [0, N]))
    src, want = _ints([0] * B), _ints([0] * B)
    k = torch.randint(0, 120, (N, Hkv, block, D), generator=g, dtype=torch.uint8).to(DEV)
    v = torch.randint(0, 120, (N, Hkv, block, D), generator=g, dtype=torch.uint8).to(DEV)
    ks, vs = torch.rand(N, Hkv, generator=g).to(DEV), torch.rand(N, Hkv, generator=g).to(DEV)

    def step():
        a, copies, lens, st = dominus_ultra_paged_fork(t, ln, src, want, ring, state, block)
        dominus_ultra_paged_copy(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), ks, vs, copies)
        a, moves, r, st = dominus_ultra_paged_compact(a, lens, ring, st, block)
        dominus_ultra_paged_copy(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), ks, vs, moves)
        for to, new in ((t, a), (ln, lens), (ring, r), (state, st)):
            to.copy_(new)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    torch.cuda.synchronize()
    # requests' rows of their own, then forks between them
    table = torch.randperm(N, generator=g)[: B * width].reshape(B, width).tolist()
    lens = [int(x) for x in torch.randint(1, width * block + 1, (B,), generator=g)]
    table = [r[: plain.pages(n, block)] + [-1] * (width - plain.pages(n, block)) for r, n in zip(table, lens)]
    held = {x for r in table for x in r if x >= 0}
    free = [x for x in range(N) if x not in held]
    rg, st = free + [-1] * (N - len(free)), [0, len(free)]
    for to, new in ((t, table), (ln, lens), (ring, rg), (state, st)):
        to.copy_(_ints(new))
    wk, wv, wks, wvs = k.clone(), v.clone(), ks.clone(), vs.clone()
    for _ in range(6):
        s = torch.randint(0, B, (B,), generator=g).tolist()
        w = [int(torch.randint(0, lens[x] + 1, (1,), generator=g)) for x in s]
        src.copy_(_ints(s))
        want.copy_(_ints(w))
        graph.replay()
        table, pairs, lens, st = plain.fork(table, lens, s, w, rg, st, block)
        for first, pair in ((True, pairs), (False, None)):
            if not first:
                table, pair, rg, st = plain.compact(table, lens, rg, st, block)
            for a, b in pair:
                if a >= 0:
                    for x in (wk, wv, wks, wvs):
                        x[b] = x[a]
        assert t.tolist() == table and ln.tolist() == lens and ring.tolist() == rg and state.tolist() == st
        for x, y in ((k, wk), (v, wv), (ks, wks), (vs, wvs)):
            assert torch.equal(x, y)


def test_on_another_stream_than_the_tensors():
    t, ln, ring, state = (_ints(x) for x in ([[0, 1], [2, -1]], [20, 7], [3, 4, -1, -1, -1], [0, 2]))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(20):
            a, copies, lens, st = dominus_ultra_paged_fork(t, ln, _ints([0, 0]), _ints([20, 20]), ring, state, 16)
            b, moves, r, s2 = dominus_ultra_paged_compact(a, lens, ring, st, 16)
    stream.synchronize()
    assert a.tolist() == [[0, 1], [0, 3]] and copies.tolist() == [[-1, -1], [1, 3]] and st.tolist() == [1, 2]
    assert b.tolist() == [[0, 1], [0, 2]] and moves.tolist() == [[3, 2], [-1, -1]] and r.tolist() == [3, 4, -1, -1, -1]
