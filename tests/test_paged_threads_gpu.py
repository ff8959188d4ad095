"""Calls that use a stream's scratch from several host threads on one stream (GPU)."""

from __future__ import annotations

import threading

import pytest
import torch

from dominusultra_b200 import _lib, dominus_ultra_decode_paged, dominus_ultra_paged_compact
from tests.test_paged_blocks_gpu import _batch, _ints
from tests.test_paged_extend_gpu import BF, HF, _call, _case

pytestmark = pytest.mark.gpu


def _compaction(seed):
    block, N, B, width = 16, 3000, 40, 30
    table, lens, free = _batch(B, width, block, N, seed)
    args = [_ints(x) for x in (table, lens, free + [-1] * (N - len(free)), [0, len(free)])]
    return lambda: torch.cat([x.flatten() for x in dominus_ultra_paged_compact(*args, block)])


def _extension(*args, **kw):
    c = _case(*args, **kw)
    return lambda: _call(c)


def _decode():
    c = _case(32, 8, 128, 1, [8000], [1], 16, BF, seed=2)
    lens = _ints(c["lens"])
    return lambda: dominus_ultra_decode_paged(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], lens, c["cos"], c["sin"])


def test_from_threads_on_one_stream(cuda_device):
    _lib.read_status(reset=True)
    calls = [
        _extension(32, 8, 128, 4, [9000, 20], [4, 4], 16, BF, seed=1),
        _compaction(1),
        _extension(4, 2, 64, 200, [5000], [200], 16, HF, seed=3),
        _decode(),
        _extension(8, 2, 256, 7, [3000] * 9, [7] * 9, 32, BF, seed=4),
        _compaction(2),
    ]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        got = []
        for j in range(120):
            at = (i * 5 + j) % len(calls)
            got.append((at, calls[at]()))
            if len(got) == 12:
                bad.extend(n for n, x in got if not torch.equal(x, want[n]))
                got.clear()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    assert _lib.read_status(reset=True)[0] == 0
