"""The paged extension where a CTA has several items one after the other, on the GPU against 64 bits (the batches are
looked at in test_paged_items_cpu.py)."""

from __future__ import annotations

import pytest
import torch

from dominusultra_b200 import _lib
from tests import _paged_exact as exact
from tests import _paged_shared as plain
from tests._paged_items import UNCUT
from tests.test_paged_extend_gpu import _call, _case

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_status(cuda_device):
    _lib.read_status(reset=True)
    yield
    assert _lib.read_status(reset=True)[0] == 0, "a test left a device status"


def _finite(cache):
    x = cache.view(torch.uint8)
    return torch.where(x & 0x7F == 0x7F, 0, x).view(cache.dtype)


@pytest.mark.parametrize("busy", [False, True], ids=["alone", "beside_other_work"])
@pytest.mark.parametrize("name", UNCUT)
def test_items_one_after_the_other(name, busy):
    # (warps of a stream drift further apart while another stream's kernels use the same memory)
    Hq, Hkv, D, T, new, past, dtype = UNCUT[name]
    c = _case(Hq, Hkv, D, T, past, new, 64 if busy else 16, dtype, seed=len(new) + T + D)
    ref, bound = plain.extend(c["q"], _finite(c["k"]), _finite(c["v"]), c["ks"], c["vs"], c["table"], c["past"], c["lens"], c["cos"], c["sin"])
    tol = exact.tolerance(ref, bound, dtype)
    other, stream = torch.empty(1 << 28, dtype=torch.uint8, device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(20):
        if busy:
            with torch.cuda.stream(stream):
                other.fill_(i)
        out = _call(c)
        assert ((out.double() - ref).abs() <= tol).all()
    torch.cuda.synchronize()


@pytest.mark.parametrize("name", UNCUT)
def test_the_same_bits_every_time(name):
    Hq, Hkv, D, T, new, past, dtype = UNCUT[name]
    c = _case(Hq, Hkv, D, T, past, new, 16, dtype, seed=len(new) + T + D)
    want = _call(c)
    for _ in range(20):
        assert torch.equal(_call(c), want)


@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("T", [1, 5, 16, 33, 70])
def test_rows_that_are_not_there_have_no_say(D, T):
    """The same bits, whatever a call before left in the shared memory of rows that a request does not fill."""
    c = _case(2, 2, D, T, [700] * 40, [T] * 40, 16, torch.bfloat16, seed=D + T)
    c["q"] = c["q"] * 2.0**-6
    c["ks"] = c["ks"] * 2.0**6
    before = _case(2, 2, D, 256, [64] * 80, [256] * 80, 16, torch.bfloat16, seed=1)
    want = None
    for factor in (0.0, 1.0, 2.0**8):
        _call(dict(before, q=before["q"] * factor))
        out = _call(c)
        want = out if want is None else want
        assert torch.equal(out, want)
