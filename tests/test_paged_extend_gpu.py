"""Attention of several new tokens per request over the paged 8-bit cache on the GPU, against 64 bits
within the bound derived in tests/_paged_shared.py."""

from __future__ import annotations

import pytest
import torch

from dominusultra_b200 import (
    _lib,
    dominus_ultra_decode_paged,
    dominus_ultra_extend_paged,
    dominus_ultra_paged_copy,
    dominus_ultra_paged_fork,
    dominus_ultra_paged_tables,
    dominus_ultra_paged_write,
    precompute_rope_cos_sin,
)
from tests import _paged_exact as exact
from tests import _paged_shared as plain

pytestmark = pytest.mark.gpu

DEV = "cuda"
NAN_BYTE = 0x7F


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


def _case(Hq, Hkv, D, T, past, new, block, dtype, seed=0, width=None, spread=3):
    """Inputs of a call; whatever is behind a request's length holds NaN bytes."""
    g = _gen(seed)
    lens = [p + n for p, n in zip(past, new)]
    B = len(lens)
    width = width or max(1, max(plain.pages(n, block) for n in lens))
    table, N = plain.make_tables(g, lens, block, width)
    k, ks = plain.make_cache(g, N, Hkv, block, D, spread=spread)
    v, vs = plain.make_cache(g, N, Hkv, block, D, spread=spread)
    for b, n in enumerate(lens):
        if n % block:
            x = int(table[b, n // block])
            for c in (k, v):
                c.view(torch.uint8)[x, :, n % block :] = NAN_BYTE
    q = torch.randn(B, Hq, T, D, generator=g).to(dtype).to(DEV)
    cos, sin = precompute_rope_cos_sin(width * block, D, DEV, dtype)
    return dict(q=q, k=k, v=v, ks=ks, vs=vs, table=table, past=past, lens=lens, cos=cos, sin=sin)


def _call(c):
    return dominus_ultra_extend_paged(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], _ints(c["past"]), _ints(c["lens"]), c["cos"], c["sin"])


def _check(c, rows=None):
    out = _call(c)
    clean = [torch.where(x.view(torch.uint8) & 0x7F == NAN_BYTE, 0, x.view(torch.uint8)).view(x.dtype) for x in (c["k"], c["v"])]
    ref, bound = plain.extend(c["q"], *clean, c["ks"], c["vs"], c["table"], c["past"], c["lens"], c["cos"], c["sin"])
    off = (out.double() - ref).abs()
    tol = exact.tolerance(ref, bound, out.dtype)
    assert torch.isfinite(out).all()
    assert (off <= tol).all(), f"off by {(off / tol).max().item():.3f} of what it may be"
    for b, (p, n) in enumerate(zip(c["past"], c["lens"])):
        assert (out[b, :, n - p :] == 0).all()
    return out


BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (6, 2), (4, 1), (16, 2), (32, 1)])
@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
def test_heads(D, Hq, Hkv, dtype):
    _check(_case(Hq, Hkv, D, 5, [0, 200, 127, 1, 3], [5, 3, 1, 0, 5], 16, dtype, seed=D + Hq))


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300])
def test_rows_and_blocks(T, block):
    _check(_case(2, 1, 64, T, [0, 77, 513], [T, max(1, T - 3), T // 2], block, HF, seed=T))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T", [8, 16, 17, 40, 70, 150])
def test_many_rows(D, T):
    _check(_case(16, 2, D, T, [0, 400, 1000], [T, T - 1, T], 16, BF, seed=T + D))


@pytest.mark.parametrize("past", [[0], [1], [15], [16], [17], [127], [128], [129], [255], [256], [4095]])
def test_borders(past):
    _check(_case(4, 2, 64, 3, past, [3], 16, BF, seed=past[0]))


@pytest.mark.parametrize("past", [[0, 0, 0], [300, 5, 16]])
def test_no_new_tokens(past):
    out = _check(_case(4, 2, 64, 4, past, [0, 0, 0], 16, BF))
    assert (out == 0).all()


@pytest.mark.parametrize("Hq,Hkv,D,T,n", [(32, 8, 128, 4, 20000), (8, 8, 64, 1, 9000), (64, 8, 128, 16, 7000), (8, 1, 128, 100, 5000), (4, 2, 256, 7, 6000), (2, 2, 32, 3, 30000), (6, 2, 16, 50, 8000)])
def test_long(Hq, Hkv, D, T, n):
    _check(_case(Hq, Hkv, D, T, [n - T], [T], 16, HF, seed=n))


@pytest.mark.parametrize("Hq,Hkv,D,T", [(32, 8, 128, 4), (8, 8, 64, 9), (16, 2, 128, 33), (4, 4, 64, 300), (2, 1, 256, 20)])
def test_mixed_batch(Hq, Hkv, D, T):
    g = _gen(T)
    new = torch.randint(0, T + 1, (23,), generator=g).tolist()
    past = torch.randint(0, 1500, (23,), generator=g).tolist()
    _check(_case(Hq, Hkv, D, T, past, new, 32, BF, seed=T, width=80))


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (8, 2, 128), (2, 2, 128), (2, 1, 256), (16, 1, 32)])
def test_a_whole_prompt(Hq, Hkv, D):
    _check(_case(Hq, Hkv, D, 1111, [0, 333], [1111, 777], 64, BF, seed=D))


def test_one_request_of_many_is_long():
    _check(_case(8, 2, 64, 2, [1] * 40 + [9000] + [2] * 30, [2] * 71, 16, HF, width=600))


def test_table_that_is_wider_than_the_lengths():
    _check(_case(8, 2, 64, 7, [30, 100], [7, 7], 16, BF, width=1000))


@pytest.mark.parametrize("T", [2, 100])
def test_scales_far_apart(T):
    # blocks whose keys' or values' scales differ by far more than the 16-bit types hold
    c = _case(4, 2, 64, T, [500, 200], [T, T], 16, HF, seed=9)
    c["q"] = c["q"] * 0.25
    for b, n in enumerate(c["lens"]):
        for i in range(plain.pages(n, 16)):
            x = int(c["table"][b, i])
            if i % 3 == 1:
                c["vs"][x] = 2.0**-60
            if i % 4 == 2:
                c["ks"][x] = 2.0**-70
    _check(c)


@pytest.mark.parametrize("T", [2, 100])
def test_values_that_outgrow_what_has_the_weight(T):
    # the first block takes nearly all of the softmax and has tiny values: outputs are those of the rest,
    # and the sum is the first block's
    c = _case(2, 1, 64, T, [300], [T], 16, HF, seed=3, spread=0)
    first = int(c["table"][0, 0])
    c["vs"][first] = 2.0**-100
    c["ks"][first] *= 4.0
    _check(c)
    c["vs"][first] = 2.0**-20
    _check(c)
    # and the other way round
    for b, i in ((0, 3), (0, 4)):
        c["vs"][int(c["table"][b, i])] = 2.0**-110
    _check(c)


@pytest.mark.parametrize("factor", [2.0**-12, 2.0**-6, 2.0**5])
def test_sizes_of_queries(factor):
    c = _case(4, 2, 128, 6, [400], [6], 16, BF, seed=2)
    c["q"] = c["q"] * factor
    _check(c)


def test_queries_beyond_fp16():
    c = _case(4, 2, 64, 6, [400], [6], 16, BF, seed=2)
    c["q"] = c["q"] * 2.0**20
    c["ks"] = c["ks"] * 2.0**-20
    _check(c)


def test_a_tail_behind_a_sink():
    # one key takes nearly all of the weight and has values of zero
    c = _case(1, 1, 64, 3, [4000], [3], 16, HF, seed=5, spread=0)
    q = torch.zeros_like(c["q"])
    q[..., 0] = 8.0
    c["q"] = q
    c["cos"], c["sin"] = torch.ones_like(c["cos"]), torch.zeros_like(c["sin"])
    k = torch.zeros(c["k"].shape, device=DEV)
    sink = int(c["table"][0, 0])
    k[sink, :, 0, 0] = 15.0
    c["k"] = k.to(torch.float8_e4m3fn)
    c["ks"].fill_(1.0)
    c["v"].view(torch.uint8)[sink, :, 0] = 0
    n = c["lens"][0]
    c["v"].view(torch.uint8)[int(c["table"][0, n // 16]), :, n % 16 :] = NAN_BYTE
    _check(c)


def test_scores_below_any_mask_value():
    c = _case(2, 2, 64, 4, [140], [4], 16, HF, seed=7, spread=0)
    c["q"] = torch.full_like(c["q"], -200.0)
    c["cos"], c["sin"] = torch.ones_like(c["cos"]), torch.zeros_like(c["sin"])
    k = torch.full(c["k"].shape, 448.0, device=DEV).to(torch.float8_e4m3fn)
    c["k"] = k
    c["ks"].fill_(2.0**40)  # scores of about -2^69
    out = _call(c)
    ref, bound = plain.extend(c["q"], k, torch.where(c["v"].view(torch.uint8) & 0x7F == NAN_BYTE, 0, c["v"].view(torch.uint8)).view(c["v"].dtype), c["ks"], c["vs"], c["table"], c["past"], c["lens"], c["cos"], c["sin"])
    # all the scores are alike, so every weight is the same whatever the scores are off by
    v = exact.rows(torch.where(c["v"].view(torch.uint8) & 0x7F == NAN_BYTE, 0, c["v"].view(torch.uint8)).view(c["v"].dtype), c["vs"], c["table"][0].long(), c["lens"][0])
    for t in range(4):
        mean, size = v[:, : 141 + t].mean(1), v[:, : 141 + t].abs().mean(1)
        off = (out[0, :, t].double() - mean).abs()
        assert (off <= 2 * (2.0**-11 + 2.0**-14) * size + 2.0**-11 * mean.abs() + 2.0**-24).all()


def test_query_rows_that_are_not_finite_stay_alone():
    c = _case(8, 2, 64, 40, [300], [40], 16, BF, seed=8)
    clean = _call(c)
    c["q"][0, 3, 7, 5] = float("nan")
    c["q"][0, 5, 0, 1] = float("inf")
    out = _call(c)
    bad = torch.zeros(8, 40, dtype=torch.bool)
    bad[3, 7] = bad[5, 0] = True
    assert torch.isnan(out[0][bad]).all()
    assert torch.equal(out[0][~bad], clean[0][~bad])


@pytest.mark.parametrize("which", ["ks", "vs"])
@pytest.mark.parametrize("T", [6, 150])
def test_a_block_whose_scale_is_not_a_number(which, T):
    # rows that see a key of the block are NaN, the rows before it are not
    c = _case(4, 2, 64, T, [290], [T], 16, BF, seed=8)
    clean = _check(c)
    page = (290 + T // 2) // 16
    x = int(c["table"][0, page])
    c[which][x, 1] = float("nan")
    c["v"].view(torch.uint8)[x, 1] = NAN_BYTE
    c["k"].view(torch.uint8)[x, 1] = NAN_BYTE
    out = _call(c)
    seen = 290 + torch.arange(T) >= page * 16
    assert torch.equal(out[0, :2], clean[0, :2])
    assert torch.isnan(out[0, 2:][:, seen]).all() and torch.equal(out[0, 2:][:, ~seen], clean[0, 2:][:, ~seen])


@pytest.mark.parametrize("bad", [-1, 10**6, 2**31 - 1, -(2**31)])
@pytest.mark.parametrize("T", [6, 150])
def test_a_block_id_out_of_range(bad, T):
    c = _case(4, 2, 64, T, [290, 80], [T, T], 16, BF, seed=8)
    clean = _check(c)
    page = (290 + T // 2) // 16
    c["table"][0, page] = bad
    out = _call(c)
    assert _status()[:3] == [7, 0, bad % 2**32]
    seen = 290 + torch.arange(T) >= page * 16
    assert torch.isnan(out[0][:, seen]).all() and torch.equal(out[0][:, ~seen], clean[0][:, ~seen])
    assert torch.equal(out[1], clean[1])


@pytest.mark.parametrize("past,n", [(-1, 3), (10, 9), (10, 15), (1000, 1004), (2**31 - 1, 5), (0, -5)])
def test_lengths_out_of_range(past, n):
    c = _case(4, 2, 64, 4, [50, 60], [4, 4], 16, BF, seed=8, width=8)
    clean = _check(c)
    out = dominus_ultra_extend_paged(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], _ints([past, 60]), _ints([n, 64]), c["cos"], c["sin"])
    assert _status()[0] == 6
    assert (out[0] == 0).all() and torch.equal(out[1], clean[1])


def test_lengths_beyond_the_rope_tables():
    c = _case(4, 2, 64, 4, [50, 60], [4, 4], 16, BF, seed=8)
    out = dominus_ultra_extend_paged(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], _ints(c["past"]), _ints(c["lens"]), c["cos"][:60], c["sin"][:60])
    assert _status()[:3] == [6, 1, 64]
    assert (out[1] == 0).all() and (out[0] != 0).any()


def test_a_single_token_agrees_with_the_decode():
    c = _case(32, 8, 128, 1, [1, 700, 4000], [1, 1, 1], 16, HF, seed=1)
    a = _check(c).double()
    b = dominus_ultra_decode_paged(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], _ints(c["lens"]), c["cos"], c["sin"]).double()
    ref, bound = plain.extend(c["q"], *(torch.where(x.view(torch.uint8) & 0x7F == NAN_BYTE, 0, x.view(torch.uint8)).view(x.dtype) for x in (c["k"], c["v"])), c["ks"], c["vs"], c["table"], c["past"], c["lens"], c["cos"], c["sin"])
    assert ((a - b).abs() <= 2 * exact.tolerance(ref, bound, HF)).all()


def test_int64_and_host_lengths():
    c = _case(4, 2, 64, 4, [50, 60], [4, 3], 16, BF, seed=8)
    want = _call(c)
    for device in ("cpu", DEV):
        out = dominus_ultra_extend_paged(
            c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"].to(device),
            torch.tensor(c["past"], device=device), torch.tensor(c["lens"], device=device), c["cos"], c["sin"],
        ) if device == "cpu" else dominus_ultra_extend_paged(
            c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], _ints(c["past"], torch.int64), _ints(c["lens"], torch.int64), c["cos"], c["sin"]
        )
        assert torch.equal(out, want)
    far = torch.tensor([2**32 + 50, 60], device=DEV)
    out = dominus_ultra_extend_paged(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], far, far + 3, c["cos"], c["sin"])
    assert _status()[0] == 6 and (out[0] == 0).all()


def test_queries_that_are_not_aligned():
    c = _case(4, 2, 64, 4, [50, 60], [4, 3], 16, BF, seed=8)
    want = _call(c)
    flat = torch.empty(c["q"].numel() + 1, dtype=BF, device=DEV)
    flat[1:] = c["q"].flatten()
    c["q"] = flat[1:].view(c["q"].shape)
    assert torch.equal(_call(c), want)


# ----------------------------------------------------------------------- streams, captures, runs


def test_same_bits_every_time():
    c = _case(32, 8, 128, 4, [3000, 20, 700], [4, 4, 2], 16, BF, seed=1)
    want = _call(c)
    for _ in range(10):
        assert torch.equal(_call(c), want)


def test_two_streams_at_once():
    a = _case(32, 8, 128, 4, [30000], [4], 16, BF, seed=1)
    b = _case(8, 2, 64, 200, [5000], [200], 16, BF, seed=2)
    wa, wb = _call(a), _call(b)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (c, s) in enumerate(zip((a, b), streams)):
            with torch.cuda.stream(s):
                got[i].append(_call(c))
    torch.cuda.synchronize()
    assert all(torch.equal(x, wa) for x in got[0]) and all(torch.equal(x, wb) for x in got[1])


def test_captured_and_replayed_with_other_lengths():
    c = _case(16, 2, 128, 9, [600, 333], [9, 9], 16, BF, seed=1, width=64)
    past, lens = _ints(c["past"]), _ints(c["lens"])
    args = [c[x] for x in ("q", "k", "v", "ks", "vs", "table")] + [past, lens, c["cos"], c["sin"]]
    dominus_ultra_extend_paged(*args)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(dominus_ultra_extend_paged(*args))
        graphs.append(g)
    for p, n in (([600, 333], [609, 342]), ([0, 0], [9, 1]), ([100, 341], [100, 342]), ([8, 17], [17, 20])):
        past.copy_(_ints(p))
        lens.copy_(_ints(n))
        c["past"], c["lens"] = p, n
        want = _call(c)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        for o in outs:
            o.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_back_to_back_with_the_decode():
    # both use the scratch of the stream
    c = _case(32, 8, 128, 4, [9000, 20], [4, 4], 16, BF, seed=1)
    d = _case(32, 8, 128, 1, [8000], [1], 16, BF, seed=2)
    dec = lambda: dominus_ultra_decode_paged(d["q"], d["k"], d["v"], d["ks"], d["vs"], d["table"], _ints(d["lens"]), d["cos"], d["sin"])  # noqa: E731
    wc, wd = _call(c), dec()
    got = [(_call(c), dec()) for _ in range(10)]
    assert all(torch.equal(x, wc) and torch.equal(y, wd) for x, y in got)


def test_a_run_of_shared_requests():
    """Prompts in chunks, a fork of one into several, drafts of their own: every step against 64 bits."""
    g = _gen(11)
    B, Hq, Hkv, D, block, width, N = 3, 8, 2, 64, 16, 40, 90
    i32 = dict(dtype=torch.int32, device=DEV)
    table, lens = torch.full((B, width), -1, **i32), torch.zeros(B, **i32)
    ring, state = torch.arange(N, **i32), _ints([0, N])
    k8, v8 = (torch.zeros(N, Hkv, block, D, device=DEV).to(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = torch.zeros(N, Hkv, device=DEV), torch.zeros(N, Hkv, device=DEV)
    cos, sin = precompute_rope_cos_sin(width * block, D, DEV, BF)

    def step(new, T):
        nonlocal lens, state
        q, k, v = (torch.randn(B, h, T, D, generator=g).to(BF).to(DEV) for h in (Hq, Hkv, Hkv))
        past = lens
        slots, lens, state = dominus_ultra_paged_tables(table, past, past + _ints(new), ring, state, block, T)
        dominus_ultra_paged_write(k, v, k8, v8, ks, vs, slots, past, cos, sin)
        out = dominus_ultra_extend_paged(q, k8, v8, ks, vs, table, past, lens, cos, sin)
        ref, bound = plain.extend(q, k8, v8, ks, vs, table, past.tolist(), lens.tolist(), cos, sin)
        assert ((out.double() - ref).abs() <= exact.tolerance(ref, bound, BF)).all()

    def fork(sources, wanted):
        nonlocal table, lens, state
        held = [exact.rows(k8, ks, table[s, : plain.pages(w, block)].long(), w) if w else None for s, w in zip(sources, wanted)]
        table, copies, lens, state = dominus_ultra_paged_fork(table, lens, _ints(sources), _ints(wanted), ring, state, block)
        dominus_ultra_paged_copy(k8, v8, ks, vs, copies)
        assert lens.tolist() == list(wanted)
        for b, (h, w) in enumerate(zip(held, wanted)):
            assert w == 0 or torch.equal(exact.rows(k8, ks, table[b, : plain.pages(w, block)].long(), w), h)
        used = {x for r, n in zip(table.tolist(), lens.tolist()) for x in r[: plain.pages(n, block)]}
        h, c = state.tolist()
        assert sorted(used | {ring.tolist()[(h + i) % N] for i in range(c)}) == list(range(N))

    step([150, 0, 0], 150)
    step([133, 0, 0], 150)
    fork([0, 0, 0], [283, 283, 100])
    step([5, 5, 4], 5)  # drafts, different in each
    n = lens.tolist()
    fork([0, 1, 2], [n[0] - 3, n[1] - 5, n[2]])  # rejected in part
    step([70, 1, 2], 70)
    fork([2, 0, 1], [lens.tolist()[2], lens.tolist()[0], 0])
    step([3, 3, 3], 3)
    fork([0, 1, 2], [0, 0, 0])
    assert state.tolist()[1] == N
