"""Values that are not numbers in an item whose keys are cut over several CTAs: the paged extension on the GPU."""

from __future__ import annotations

import pytest
import torch

from dominusultra_b200 import _lib
from tests import _paged_items as items
from tests.test_paged_extend_gpu import NAN_BYTE, _call, _case, _check

pytestmark = pytest.mark.gpu

# new tokens of four query heads on two key heads: every layout of an item's rows (one item of a key head; at head_dim
# 256 that is up to 64 tokens)
ROWS = [1, 20, 50, 100]


@pytest.fixture(autouse=True)
def _clean_status(cuda_device):
    _lib.read_status(reset=True)
    yield
    assert _lib.read_status(reset=True)[0] == 0, "a test left a device status"


def _fragments(c, T, D):
    """Key tiles of the fragments of the first key head's only item, and the keys of a tile."""
    new = [n - p for n, p in zip(c["lens"], c["past"])]
    cut = [f for cta in items.split(c["past"], new, 4, 2, D, T) for f in cta if f[1] == 0 and f[2] == 0]
    return [(f[4], f[5]) for f in cut], items.plan(T, 2, D)[2]


@pytest.mark.parametrize("which", ["ks", "vs", "id"])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
@pytest.mark.parametrize("T", ROWS)
@pytest.mark.parametrize("D", [16, 64, 128, 256])
def test_a_fragment_without_a_number(D, T, where, which):
    """Every key of one fragment lies in a block with a scale that is not a number, or without a block id: every row that
    sees one of them is NaN, the others keep their bits."""
    n, T = 20000, min(T, 64) if D == 256 else T
    c = _case(4, 2, D, T, [n - T], [T], 128, torch.bfloat16, seed=D + T)
    clean = _check(c)
    cut, keys = _fragments(c, T, D)
    assert len(cut) >= 3 and cut[-1][1] * keys >= n
    lo, hi = cut[{"first": 0, "middle": len(cut) // 2, "last": -1}[where]]
    pages = range(lo * keys // 128, min(-(-hi * keys // 128), -(-n // 128)))
    for page in pages:
        x = int(c["table"][0, page])
        if which == "id":
            c["table"][0, page] = -1
        else:
            c[which][x, 0] = float("nan")
            for cache in (c["k"], c["v"]):
                cache.view(torch.uint8)[x, 0] = NAN_BYTE
    out = _call(c)
    status = _lib.read_status(reset=True)
    assert status[:2] == [7, 0] if which == "id" else status[0] == 0
    seen = n - T + torch.arange(T) >= pages[0] * 128
    assert seen.any()
    heads = slice(None) if which == "id" else slice(0, 2)
    assert torch.isnan(out[0, heads][:, seen]).all()
    assert torch.equal(out[0, heads][:, ~seen], clean[0, heads][:, ~seen])
    if which != "id":
        assert torch.equal(out[0, 2:], clean[0, 2:])


@pytest.mark.parametrize("cut", [False, True], ids=["whole", "cut"])
@pytest.mark.parametrize("T", ROWS)
@pytest.mark.parametrize("D", [16, 64, 128, 256])
def test_scores_that_are_all_minus_infinity(D, T, cut):
    """The softmax of a row that has no other scores is not a number, however its keys are cut."""
    n = 20000 if cut else T + 3
    c = _case(4, 2, D, T, [n - T], [T], 16, torch.float16, seed=1)
    c["cos"].fill_(0.75)
    c["sin"].fill_(0.5)
    for i in (0, D // 2):
        c["k"].view(torch.uint8)[..., i] = 0xB8  # -1 in the pair of coordinates that the infinity turns into
    clean = _call(c)
    c["q"][0, 1, 0, 0] = float("inf")
    if T > 1:
        c["q"][0, 3, T - 1, 0] = float("inf")
    out = _call(c)
    bad = torch.isinf(c["q"][0]).any(-1)
    assert torch.isfinite(clean).all()
    assert torch.isnan(out[0][bad]).all() and torch.equal(out[0][~bad], clean[0][~bad])
