"""Paged 8-bit cache on the GPU against plain 64-bit implementations (tests/_paged.py): block tables
and the writer bit for bit, the attention within the bound derived there."""

from __future__ import annotations

import pytest
import torch

from dominusultra_b200 import (
    _lib,
    dominus_ultra_decode_paged,
    dominus_ultra_paged_tables,
    dominus_ultra_paged_write,
    dominus_ultra_prefill,
    precompute_rope_cos_sin,
)
from tests import _paged as plain

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


# ----------------------------------------------------------------------------------------- tables


def _check_tables(old, new, ring, state, width, block, max_new, table=None, seed=0, cpu_lens=False):
    g = _gen(seed)
    B = len(old)
    if table is None:
        table = torch.randint(0, len(ring), (B, width), generator=g).tolist()
    t_dev = torch.tensor(table, dtype=torch.int32, device=DEV)
    r_dev = torch.tensor(ring, dtype=torch.int32, device=DEV)
    s_dev = torch.tensor(state, dtype=torch.int32, device=DEV)
    lens = [torch.tensor(x, dtype=torch.int32, device="cpu" if cpu_lens else DEV) for x in (old, new)]
    got = dominus_ultra_paged_tables(t_dev, *lens, r_dev, s_dev, block, max_new)
    want = plain.tables(table, list(old), list(new), ring, list(state), block, max_new)
    assert got[0].tolist() == want[0]
    assert got[1].tolist() == want[1]
    assert got[2].tolist() == want[2]
    assert t_dev.tolist() == table and r_dev.tolist() == ring and s_dev.tolist() == list(state)


@pytest.mark.parametrize("B,T,block", [(1, 1, 16), (3, 1, 128), (64, 1, 16), (5, 777, 32), (511, 7, 64), (513, 33, 16), (1030, 2, 32)])
@pytest.mark.parametrize("short", [False, True])
def test_tables(B, T, block, short):
    g = _gen(B * 7 + T)
    width = plain.pages(2 * T + 300, block)
    cap = width * block
    old = torch.randint(0, cap - T + 1, (B,), generator=g)
    kind = torch.randint(0, 4, (B,), generator=g)
    grow = torch.randint(1, T + 1, (B,), generator=g)
    new = torch.where(kind == 0, torch.zeros_like(old), torch.where(kind == 1, old // 2, old + grow))
    old, new = old.tolist(), new.tolist()
    held = sum(plain.pages(n, block) for n in old)
    need = sum(max(0, plain.pages(w, block) - plain.pages(o, block)) for o, w in zip(old, new))
    N = held + need + 3
    ring = torch.randperm(N, generator=g).tolist()
    _check_tables(old, new, ring, [N - 2, need // 2 if short else need], width, block, T, cpu_lens=B == 3)


def test_tables_without_new_tokens():
    _check_tables([20, 5], [0, 5], [0, 1, 2, 3, 4, 5], [4, 1], 2, 16, 0)


def test_tables_at_capacity_and_int64():
    t = torch.full((2, 4), -1, dtype=torch.int32, device=DEV)
    ring = torch.arange(9, dtype=torch.int32, device=DEV)
    state = torch.tensor([0, 9], dtype=torch.int32, device=DEV)
    old = torch.zeros(2, dtype=torch.int64, device=DEV)
    slots, lens, left = dominus_ultra_paged_tables(t, old, old + 64, ring, state, 16, 64)
    assert lens.tolist() == [64, 64] and left.tolist() == [8, 1]
    assert slots.flatten().tolist() == list(range(128))
    # int64 lengths beyond int32 leave the request alone
    _, lens, _ = dominus_ultra_paged_tables(t, lens.long(), torch.tensor([2**32, 64], device=DEV), ring, left, 16, 64)
    assert lens.tolist() == [64, 64] and _status()[:2] == [6, 0]


@pytest.mark.parametrize("old,new", [([-1, 5], [3, 6]), ([5, 5], [6, 500]), ([5, 5], [6, -3]), ([500, 5], [5, 6]), ([5, 0], [6, 12])])
def test_tables_lengths_out_of_range(old, new):
    _check_tables(old, new, list(range(40)), [3, 30], 4, 16, 8)
    assert _status()[0] == 6


@pytest.mark.parametrize("state", [[-1, 4], [8, 4], [0, 9], [0, -2], [0, 8]])
def test_tables_ring_state_out_of_range(state):
    # (the last: more given back than the ring has room for)
    _check_tables([40, 8], [0, 9], list(range(8)), state, 4, 16, 1)
    assert _status()[0] == 7


def test_tables_damaged_entry_gives_no_slot():
    t = torch.tensor([[99, 0], [1, 0]], dtype=torch.int32, device=DEV)
    ring, state = torch.arange(4, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    lens = torch.tensor([3, 4], dtype=torch.int32, device=DEV)
    slots, _, _ = dominus_ultra_paged_tables(t, lens, lens + 1, ring, state, 16, 1)
    assert slots.tolist() == [[-1], [20]] and _status()[:3] == [7, 0, 99]


# ------------------------------------------------------------------------------------------ write


def _write_case(B, Hkv, D, T, block, past, counts, dtype, seed, scale_up=1.0):
    """Random cache and new rows; slots over distinct blocks from scattered ids."""
    g = _gen(seed)
    width = plain.pages(block - 1 + T, block)
    N = B * width + 2
    ids = torch.randperm(N, generator=g)[: B * width].reshape(B, width)
    slots = torch.full((B, T), -1, dtype=torch.int32)
    for b in range(B):
        for t in range(counts[b]):
            pg, r = divmod(past[b] % block + t, block)
            slots[b, t] = int(ids[b, pg]) * block + r
    x = lambda: plain.quantise_cache(torch.randn(N, Hkv, block, D, generator=g).double())  # noqa: E731
    (k8, ks), (v8, vs) = x(), x()
    size = torch.exp2(torch.randint(-3, 4, (B, Hkv, 1, 1), generator=g).float()) * scale_up
    kn = (torch.randn(B, Hkv, T, D, generator=g) * size).to(dtype)
    vn = (torch.randn(B, Hkv, T, D, generator=g) * size).to(dtype)
    cos, sin = precompute_rope_cos_sin(max(past) + T, D, "cpu", dtype)
    return kn, vn, k8, v8, ks, vs, slots, cos, sin


def _run_write(kn, vn, k8, v8, ks, vs, slots, past, cos, sin):
    d = lambda t: t.to(DEV)  # noqa: E731
    k8d, v8d = d(k8.float().to(torch.float8_e4m3fn)), d(v8.float().to(torch.float8_e4m3fn))
    ksd, vsd = d(ks.float()), d(vs.float())
    dominus_ultra_paged_write(d(kn), d(vn), k8d, v8d, ksd, vsd, d(slots), torch.tensor(past, dtype=torch.int32, device=DEV), d(cos), d(sin))
    return [t.cpu().double() for t in (k8d, v8d, ksd, vsd)]


def _same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=1e9), torch.nan_to_num(b, nan=1e9))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Hkv,D,T,block,past,counts", [
    (1, 1, 16, 1, 16, [0], [1]),
    (3, 2, 64, 1, 16, [15, 16, 1000], [1, 1, 0]),
    (4, 8, 128, 1, 128, [127, 0, 5, 300], [1, 1, 1, 1]),
    (2, 3, 128, 37, 16, [5, 0], [37, 20]),
    (2, 2, 256, 130, 128, [100, 0], [130, 129]),
    (3, 1, 32, 70, 64, [63, 1, 64], [70, 1, 64]),
    (2, 4, 64, 200, 32, [31, 17], [200, 0]),
    (1, 2, 16, 260, 128, [7], [259]),
    # each number of warps and rows per thread that an item can take
    (2, 2, 16, 70, 32, [3, 0], [70, 33]),
    (3, 5, 64, 50, 16, [15, 0, 8], [50, 16, 49]),
    (3, 3, 128, 90, 32, [31, 0, 40], [90, 31, 64]),
    (2, 3, 128, 150, 64, [5, 64], [150, 64]),
    (2, 1, 128, 300, 128, [127, 1], [300, 128]),
    (2, 2, 256, 40, 16, [0, 9], [40, 23]),
])
def test_write(B, Hkv, D, T, block, past, counts, dtype):
    c = _write_case(B, Hkv, D, T, block, past, counts, dtype, B + D + T)
    kn, vn, k8, v8, ks, vs, slots, cos, sin = c
    got = _run_write(kn, vn, k8, v8, ks, vs, slots, past, cos, sin)
    plain.write(kn, vn, k8, v8, ks, vs, slots.tolist(), past, cos, sin)
    for name, a, w in zip(("k8", "v8", "ks", "vs"), got, (k8, v8, ks, vs)):
        assert _same(a, w), name


def test_write_rounds_the_exact_sum_once():
    """Rotations whose exact value lies just beside a tie between two e4m3 values, where a sum rounded
    to 32 bits first falls on the tie: fp16 keys 1 + j 2^-10 against tables of small sines."""
    D, T, block = 16, 128, 128
    g = _gen(11)
    kn = (1 + torch.randint(0, 1024, (1, 1, T, D), generator=g).double() / 1024).half()
    kn[..., D // 2 :] = torch.exp2(torch.randint(-14, -6, (1, 1, T, D // 2), generator=g).double()).half()
    cos = torch.ones(T, D // 2, dtype=torch.float16)
    sin = torch.exp2(-torch.randint(8, 15, (T, D // 2), generator=g).double()).half()
    # values 1.0625, 1.1875, ...: ties of e4m3 at the unit that amax gives
    kn[..., : D // 2] = (1 + (2 * torch.randint(0, 8, (1, 1, T, D // 2), generator=g).double() + 1) / 16).half()
    k8 = torch.zeros(1, 1, block, D, dtype=torch.float64)
    z = lambda: torch.zeros(1, 1, dtype=torch.float64)  # noqa: E731
    slots = torch.arange(T, dtype=torch.int32)[None]
    got = _run_write(kn, kn, k8, k8.clone(), z(), z(), slots, [0], cos, sin)
    want = [k8.clone(), k8.clone(), z(), z()]
    plain.write(kn, kn, *want, slots.tolist(), [0], cos, sin)
    for a, w in zip(got, want):
        assert _same(a, w)


def test_write_zero_rows_and_growth_from_zero():
    """All-zero rows take the smallest scale; a later row makes it grow and the zeros stay zeros."""
    kn = torch.zeros(1, 1, 3, 32, dtype=torch.bfloat16)
    c = _write_case(1, 1, 32, 1, 16, [3], [1], torch.bfloat16, 2)
    k8 = torch.zeros(1, 1, 16, 32, dtype=torch.float64)
    z = torch.zeros(1, 1, dtype=torch.float64)
    cos, sin = precompute_rope_cos_sin(8, 32, "cpu", torch.bfloat16)
    k8a, v8a, ksa, vsa = _run_write(kn, kn, k8, k8.clone(), z, z.clone(), torch.tensor([[0, 1, 2]], dtype=torch.int32), [0], cos, sin)
    assert ksa.item() == 2.0**-64 and vsa.item() == 2.0**-64 and k8a.abs().max() == 0
    got = _run_write(c[0], c[1], k8a, v8a, ksa, vsa, torch.tensor([[3]], dtype=torch.int32), [3], cos, sin)
    plain.write(c[0], c[1], k8a, v8a, ksa, vsa, [[3]], [3], cos, sin)
    for a, w in zip(got, (k8a, v8a, ksa, vsa)):
        assert _same(a, w)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_write_not_finite_marks_its_block_only(bad):
    past, counts = [0, 4], [20, 5]
    c = _write_case(2, 2, 64, 20, 16, past, counts, torch.bfloat16, 9)
    kn, vn, k8, v8, ks, vs, slots, cos, sin = c
    kn[0, 1, 17, 3] = bad
    vn[1, 0, 2, 60] = bad
    got = _run_write(kn, vn, k8, v8, ks, vs, slots, past, cos, sin)
    plain.write(kn, vn, k8, v8, ks, vs, slots.tolist(), past, cos, sin)
    for a, w in zip(got, (k8, v8, ks, vs)):
        assert _same(a, w)
    assert got[2].isnan().sum() == 1 and got[3].isnan().sum() == 1


def test_write_damaged_slots_are_skipped():
    past, counts = [3, 0, 0], [2, 2, 2]
    c = _write_case(3, 1, 64, 2, 16, past, counts, torch.bfloat16, 4)
    kn, vn, k8, v8, ks, vs, slots, cos, sin = c
    N = k8.shape[0]
    slots[0, 0] += 1                   # not where position 3 belongs
    slots[1, :] += N * 16              # beyond the cache
    got = _run_write(kn, vn, k8, v8, ks, vs, slots, past, cos, sin)
    assert _status()[0] == 7
    slots[:2] = -1
    plain.write(kn, vn, k8, v8, ks, vs, slots.tolist(), past, cos, sin)
    for a, w in zip(got, (k8, v8, ks, vs)):
        assert _same(a, w)


@pytest.mark.parametrize("T,block,past", [(5, 16, 3), (40, 16, 3), (140, 128, 0), (6, 64, 0)])
def test_write_slots_behind_a_row_without_one_are_reported(T, block, past):
    """A block's new rows start with its first token; slots behind a hole there are not written."""
    c = _write_case(2, 2, 64, T, block, [past, past], [T, T], torch.bfloat16, 12)
    kn, vn, k8, v8, ks, vs, slots, cos, sin = c
    t0 = 0 if T <= block else block - past  # the first token of the request's first or second block
    n = min(T - t0, block)
    slots[1, t0] = -1
    got = _run_write(kn, vn, k8, v8, ks, vs, slots, [past, past], cos, sin)
    assert _status()[:2] == [7, 1]
    slots[1, t0 : t0 + n] = -1
    plain.write(kn, vn, k8, v8, ks, vs, slots.tolist(), [past, past], cos, sin)
    for a, w in zip(got, (k8, v8, ks, vs)):
        assert _same(a, w)


def test_write_positions_beyond_the_rope_tables():
    past = [14]
    c = _write_case(1, 1, 64, 4, 16, past, [4], torch.bfloat16, 6)
    kn, vn, k8, v8, ks, vs, slots, cos, sin = c
    got = _run_write(kn, vn, k8, v8, ks, vs, slots, past, cos[:17], sin[:17])
    assert _status()[:3] == [6, 0, 17]
    same = _run_write(kn, vn, k8, v8, ks, vs, slots, [-2], cos, sin)
    assert _status()[0] == 6
    for a, w in zip(same, (k8, v8, ks, vs)):
        assert _same(a, w)
    slots[0, 3:] = -1  # the token at position 17, of keys and values both
    plain.write(kn, vn, k8, v8, ks, vs, slots.tolist(), past, cos, sin)
    for a, w in zip(got, (k8, v8, ks, vs)):
        assert _same(a, w)


def test_write_of_nothing_leaves_everything():
    """Tokens beyond the tables in a fresh block: neither rows nor scales change."""
    past = [16]
    c = _write_case(1, 2, 64, 4, 16, past, [4], torch.bfloat16, 6)
    kn, vn, k8, v8, ks, vs, slots, cos, sin = c
    got = _run_write(kn, vn, k8, v8, ks, vs, slots, past, cos[:16], sin[:16])
    assert _status()[0] == 6
    for a, w in zip(got, (k8, v8, ks, vs)):
        assert _same(a, w)


# ----------------------------------------------------------------------------------------- attend


def _attend_case(B, Hq, Hkv, D, block, lens, dtype, seed, spread=1.0):
    g = _gen(seed)
    width = max(1, plain.pages(max(lens), block))
    N = sum(plain.pages(n, block) for n in lens) + 2
    perm = torch.randperm(N, generator=g).tolist()
    table, at = [], 0
    for n in lens:
        m = plain.pages(n, block)
        table.append(perm[at : at + m] + [-1 - 7 * i for i in range(width - m)])
        at += m
    size = torch.exp2(torch.randint(-3, 3, (N, Hkv, 1, 1), generator=g).double())
    k8, ks = plain.quantise_cache(torch.randn(N, Hkv, block, D, generator=g).double() * spread)
    v8, vs = plain.quantise_cache(torch.randn(N, Hkv, block, D, generator=g).double() * size)
    q = torch.randn(B, Hq, 1, D, generator=g).to(dtype)
    cos, sin = precompute_rope_cos_sin(max(1, max(lens)), D, "cpu", dtype)
    return q, k8, v8, ks, vs, table, cos, sin


def _to_cache(x8, table, lens, block):
    """e4m3 bytes on the GPU with every row that is not a cached token's NaN."""
    used = torch.zeros(x8.shape[0], block, dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(plain.pages(n, block)):
            used[table[b][i], : min(block, n - i * block)] = True
    x = x8.float().to(torch.float8_e4m3fn).view(torch.uint8)
    x = torch.where(used[:, None, :, None], x, torch.tensor(NAN_BYTE, dtype=torch.uint8))
    return x.to(DEV).view(torch.float8_e4m3fn)


def _scales(s, table, lens, block):
    used = sorted({table[b][i] for b, n in enumerate(lens) for i in range(plain.pages(n, block))})
    x = torch.full_like(s, float("nan"))
    x[used] = s[used]
    return x.float().to(DEV)


def _check_attend(B, Hq, Hkv, D, block, lens, dtype, seed=0, spread=1.0):
    q, k8, v8, ks, vs, table, cos, sin = _attend_case(B, Hq, Hkv, D, block, lens, dtype, seed, spread)
    got = dominus_ultra_decode_paged(
        q.to(DEV), _to_cache(k8, table, lens, block), _to_cache(v8, table, lens, block), _scales(ks, table, lens, block),
        _scales(vs, table, lens, block), torch.tensor(table, dtype=torch.int32, device=DEV),
        torch.tensor(lens, dtype=torch.int32, device=DEV), cos.to(DEV), sin.to(DEV),
    ).cpu()
    want, bound = plain.attend(q, k8, v8, ks, vs, table, lens, cos, sin)
    off = (got.double() - want).abs()
    tol = plain.tolerance(want, bound, dtype)
    assert got.shape == want.shape and got.dtype == dtype
    assert bool((off <= tol).all()), f"worst {(off / tol).max():.3f} of the tolerance"


HEADS = [(1, 1, 16), (2, 2, 32), (8, 8, 64), (6, 2, 64), (4, 1, 128), (8, 2, 128), (16, 2, 128), (5, 1, 128), (24, 2, 64), (32, 1, 64), (4, 2, 256), (16, 1, 256), (12, 4, 32), (6, 3, 16), (1, 1, 128), (2, 2, 256), (8, 1, 32), (8, 1, 16), (2, 1, 16), (7, 1, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
def test_attend_heads(Hq, Hkv, D, dtype):
    _check_attend(4, Hq, Hkv, D, 16, [1, 16, 131, 700], dtype, seed=Hq + D)


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (3, 3, 64), (2, 1, 256), (2, 1, 16)])
def test_attend_blocks(block, Hq, Hkv, D):
    lens = [block - 1, block, block + 1, 127, 128, 129, 0, 1000]
    _check_attend(8, Hq, Hkv, D, block, lens, torch.bfloat16, seed=block)


@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 3], [4096], [8191, 1], [5, 4, 3, 2, 1, 0, 250, 260, 2000], [256] * 40, [130, 1] * 80])
@pytest.mark.parametrize("Hq,Hkv,D,block", [(4, 1, 128, 16), (2, 2, 64, 64)])
def test_attend_lengths(lens, Hq, Hkv, D, block):
    _check_attend(len(lens), Hq, Hkv, D, block, lens, torch.float16, seed=len(lens) + D)


def test_attend_sharp_scores():
    """Scores that differ by hundreds: the running maximum moves often."""
    _check_attend(3, 8, 2, 128, 32, [900, 1500, 60], torch.bfloat16, seed=3, spread=12.0)
    _check_attend(3, 4, 4, 64, 16, [900, 1500, 60], torch.float16, seed=4, spread=12.0)


def test_attend_rising_scores():
    """Every key scores above the ones before it."""
    D, block, n = 128, 16, 1000
    q = torch.zeros(1, 4, 1, D, dtype=torch.float16)
    q[..., 0] = 8.0
    k = torch.zeros(plain.pages(n, block), 1, block, D, dtype=torch.float64)
    k.view(-1, D)[:n, 0] = torch.linspace(-40, 40, n).double()
    k8, ks = plain.quantise_cache(k)
    v8, vs = plain.quantise_cache(torch.randn(k.shape, generator=_gen(1)).double())
    cos, sin = torch.ones(n, D // 2, dtype=torch.float16), torch.zeros(n, D // 2, dtype=torch.float16)
    table = [list(range(k.shape[0]))]
    d = lambda t, dt=torch.float8_e4m3fn: t.float().to(dt).to(DEV)  # noqa: E731
    got = dominus_ultra_decode_paged(q.to(DEV), d(k8), d(v8), d(ks, torch.float32), d(vs, torch.float32), torch.tensor(table, dtype=torch.int32, device=DEV), torch.tensor([n], dtype=torch.int32, device=DEV), cos.to(DEV), sin.to(DEV)).cpu()
    want, bound = plain.attend(q, k8, v8, ks, vs, table, [n], cos, sin)
    assert bool(((got.double() - want).abs() <= plain.tolerance(want, bound, torch.float16)).all())


def test_attend_huge_negative_scores():
    """Every score is far below any usual mask value; the largest still carries the weight."""
    D, block, n = 64, 16, 40
    q = torch.full((1, 2, 1, D), 2.0**60, dtype=torch.bfloat16)
    k = -torch.ones(3, 2, block, D, dtype=torch.float64)
    k[1, :, 3] = -0.5
    k8, ks = plain.quantise_cache(k)
    ks = ks * 2.0**50
    v8, vs = plain.quantise_cache(torch.randn(k.shape, generator=_gen(1)).double())
    cos, sin = torch.ones(n, D // 2, dtype=torch.bfloat16), torch.zeros(n, D // 2, dtype=torch.bfloat16)
    table = [[0, 1, 2]]
    d = lambda t, dt=torch.float8_e4m3fn: t.float().to(dt).to(DEV)  # noqa: E731
    got = dominus_ultra_decode_paged(q.to(DEV), d(k8), d(v8), d(ks, torch.float32), d(vs, torch.float32), torch.tensor(table, dtype=torch.int32, device=DEV), torch.tensor([n], dtype=torch.int32, device=DEV), cos.to(DEV), sin.to(DEV)).cpu()
    want = (v8[1, :, 3] * vs[1, :, None])[None, :, None]  # one key takes all
    # the value is carried to 2^-11 (parts of the weight) and rounded to half a step
    assert bool(((got.double() - want).abs() <= want.abs() * (2.0**-8 + 2.0**-10) + 1e-30).all())


def _simple_call(B=2, Hq=4, Hkv=2, D=64, block=16, lens=(40, 100), dtype=torch.bfloat16, seed=1):
    q, k8, v8, ks, vs, table, cos, sin = _attend_case(B, Hq, Hkv, D, block, list(lens), dtype, seed)
    args = [q.to(DEV), k8.float().to(torch.float8_e4m3fn).to(DEV), v8.float().to(torch.float8_e4m3fn).to(DEV), ks.float().to(DEV),
            vs.float().to(DEV), torch.tensor(table, dtype=torch.int32, device=DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
            cos.to(DEV), sin.to(DEV)]
    return args


def test_attend_lengths_out_of_range():
    a = _simple_call()
    good = dominus_ultra_decode_paged(*a)
    for bad in (-1, a[5].shape[1] * 16 + 1, 101):
        a[6] = torch.tensor([40, bad], dtype=torch.int32, device=DEV)
        out = dominus_ultra_decode_paged(*a)
        assert torch.equal(out[0], good[0]) and out[1].abs().max() == 0
        assert _status()[:3] == [6, 1, bad & 0xFFFFFFFF]


@pytest.mark.parametrize("page", [0, 3, 6])
@pytest.mark.parametrize("value", [-1, 10**6, -(2**31)])
def test_attend_bad_page(page, value):
    a = _simple_call()
    good = dominus_ultra_decode_paged(*a)
    a[5][1, page] = value
    out = dominus_ultra_decode_paged(*a)
    assert torch.equal(out[0], good[0]) and bool(out[1].isnan().all())
    assert _status()[:3] == [7, 1, value & 0xFFFFFFFF]


def test_attend_nan_scale_reaches_its_heads_only():
    a = _simple_call()
    good = dominus_ultra_decode_paged(*a)
    for which in (3, 4):
        b = list(a)
        b[which] = a[which].clone()
        b[which][a[5][0, 1].item(), 1] = float("nan")
        out = dominus_ultra_decode_paged(*b)
        assert bool(out[0, 2:].isnan().all()) and torch.equal(out[0, :2], good[0, :2]) and torch.equal(out[1], good[1])


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 1, 64), (16, 2, 128), (6, 2, 32), (4, 4, 256), (4, 1, 16)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attend_query_not_finite_reaches_its_head_only(Hq, Hkv, D, bad):
    a = _simple_call(B=2, Hq=Hq, Hkv=Hkv, D=D, lens=(40, 300))
    good = dominus_ultra_decode_paged(*a)
    b = list(a)
    b[0] = a[0].clone()
    b[0][1, Hq - 2, 0, D - 3] = bad
    out = dominus_ultra_decode_paged(*b)
    assert bool(out[1, Hq - 2].isnan().all()) and torch.equal(out[0], good[0])
    others = [h for h in range(Hq) if h != Hq - 2]
    assert torch.equal(out[1, others], good[1, others])


def test_attend_on_the_host_checked():
    a = _simple_call()
    good = dominus_ultra_decode_paged(*a)
    b = list(a)
    b[5], b[6] = a[5].cpu(), a[6].cpu()
    assert torch.equal(dominus_ultra_decode_paged(*b), good)
    b[5] = b[5].clone()
    b[5][1, 2] = -1
    with pytest.raises(ValueError, match=r"block_table\[1, 2\]"):
        dominus_ultra_decode_paged(*b)
    b[6] = torch.tensor([40, 101])
    with pytest.raises(ValueError, match=r"cache_seqlens\[1\] = 101"):
        dominus_ultra_decode_paged(*b)


def test_attend_repeats_bit_for_bit_and_on_other_streams():
    a = _simple_call(B=3, Hq=8, Hkv=1, D=128, lens=(3000, 100, 2500))
    first = dominus_ultra_decode_paged(*a)
    for _ in range(20):
        assert torch.equal(dominus_ultra_decode_paged(*a), first)
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    outs = []
    for i in range(40):
        with torch.cuda.stream(streams[i % 4]):
            outs.append(dominus_ultra_decode_paged(*a))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)


def test_attend_unaligned_query_view():
    a = _simple_call(B=1, lens=(77,))
    good = dominus_ultra_decode_paged(*a)
    buf = torch.empty(a[0].numel() + 1, dtype=a[0].dtype, device=DEV)
    view = buf[1:].view(a[0].shape)
    view.copy_(a[0])
    a[0] = view
    assert torch.equal(dominus_ultra_decode_paged(*a), good)


def test_attend_offsets_beyond_32_bits():
    """A cache of over 2^32 bytes, the request's blocks at its far end."""
    N, Hkv, block, D, n = 36000, 8, 128, 128, 300
    assert N * Hkv * block * D > 2**32
    q, k8, v8, ks, vs, table, cos, sin = _attend_case(1, 16, Hkv, D, block, [n], torch.bfloat16, 8)
    k = torch.zeros(N, Hkv, block, D, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    v = torch.zeros(N, Hkv, block, D, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    kss, vss = torch.ones(N, Hkv, device=DEV), torch.ones(N, Hkv, device=DEV)
    far = [N - 1 - 2 * i for i in range(len(table[0]))]
    for i, blk in enumerate(far):
        k.view(torch.uint8)[blk] = k8[table[0][i]].float().to(torch.float8_e4m3fn).view(torch.uint8).to(DEV)
        v.view(torch.uint8)[blk] = v8[table[0][i]].float().to(torch.float8_e4m3fn).view(torch.uint8).to(DEV)
        kss[blk], vss[blk] = ks[table[0][i]].float().to(DEV), vs[table[0][i]].float().to(DEV)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    t = torch.tensor([far], dtype=torch.int32, device=DEV)
    got = dominus_ultra_decode_paged(q.to(DEV), k, v, kss, vss, t, lens, cos.to(DEV), sin.to(DEV)).cpu()
    want, bound = plain.attend(q, k8, v8, ks, vs, table, [n], cos, sin)
    assert bool(((got.double() - want).abs() <= plain.tolerance(want, bound, torch.bfloat16)).all())
    # the writer reaches the same far block
    past, T = 5, 1
    kn = torch.randn(1, Hkv, T, D, generator=_gen(2)).bfloat16()
    slots = torch.tensor([[far[0] * block + past]], dtype=torch.int32)
    w = [k[far[0]][None].cpu().double(), v[far[0]][None].cpu().double(), kss[far[0]][None].cpu().double(), vss[far[0]][None].cpu().double()]
    dominus_ultra_paged_write(kn.to(DEV), kn.to(DEV), k, v, kss, vss, slots.to(DEV), torch.tensor([past], dtype=torch.int32, device=DEV), cos.to(DEV), sin.to(DEV))
    plain.write(kn, kn, *w, [[past]], [past], cos, sin)
    for a, b in zip((k[far[0]], v[far[0]], kss[far[0]], vss[far[0]]), w):
        assert torch.equal(a.cpu().double(), b[0])


# ----------------------------------------------------------------------------------- together


class _Loop:
    """A cache with its bookkeeping on the GPU, and the same step in plain 64-bit form."""

    def __init__(self, B, Hq, Hkv, D, block, width, N, dtype):
        self.B, self.Hq, self.Hkv, self.D, self.block, self.dtype = B, Hq, Hkv, D, block, dtype
        i32 = dict(dtype=torch.int32, device=DEV)
        garbage = lambda: torch.full((N, Hkv, block, D), NAN_BYTE, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)  # noqa: E731
        self.k, self.v = garbage(), garbage()
        self.ks, self.vs = torch.zeros(N, Hkv, device=DEV), torch.zeros(N, Hkv, device=DEV)
        self.table = torch.full((B, width), -1, **i32)
        self.ring, self.state = torch.arange(N, **i32), torch.tensor([0, N], **i32)
        self.lens = torch.zeros(B, **i32)
        cos, sin = precompute_rope_cos_sin(width * block, D, "cpu", dtype)
        self.cos, self.sin, self.cos_c, self.sin_c = cos.to(DEV), sin.to(DEV), cos, sin
        self.p_table, self.p_ring, self.p_state, self.p_lens = [[-1] * width for _ in range(B)], list(range(N)), [0, N], [0] * B
        z = lambda: torch.zeros(N, Hkv, block, D, dtype=torch.float64)  # noqa: E731
        self.p = [z(), z(), torch.zeros(N, Hkv, dtype=torch.float64), torch.zeros(N, Hkv, dtype=torch.float64)]

    def step(self, want, q, kn, vn):
        """want: new lengths on the GPU; q [B, Hq, 1, D], kn, vn [B, Hkv, T, D]."""
        slots, lens, state = dominus_ultra_paged_tables(self.table, self.lens, want, self.ring, self.state, self.block, kn.shape[2])
        dominus_ultra_paged_write(kn, vn, self.k, self.v, self.ks, self.vs, slots, self.lens, self.cos, self.sin)
        out = dominus_ultra_decode_paged(q, self.k, self.v, self.ks, self.vs, self.table, lens, self.cos, self.sin)
        self.lens.copy_(lens)
        self.state.copy_(state)
        return out

    def plain_step(self, want, q, kn, vn):
        old = list(self.p_lens)
        slots, self.p_lens, self.p_state = plain.tables(self.p_table, old, want, self.p_ring, self.p_state, self.block, kn.shape[2])
        plain.write(kn, vn, *self.p, slots, old, self.cos_c, self.sin_c)
        return plain.attend(q, *self.p, self.p_table, self.p_lens, self.cos_c, self.sin_c)


@pytest.mark.parametrize("Hq,Hkv,D,block,dtype", [(8, 2, 128, 16, torch.bfloat16), (2, 2, 64, 32, torch.float16)])
def test_generation_loop_with_turnover(Hq, Hkv, D, block, dtype):
    """Prompts, single tokens, rejected tokens, ends and beginnings, with blocks running short."""
    B, width, N = 5, 160 // block, 30 * 16 // block
    loop = _Loop(B, Hq, Hkv, D, block, width, N, dtype)
    g = _gen(17)
    for step in range(14):
        T = 45 if step % 5 == 0 else 1
        lens = loop.p_lens
        want = []
        for b in range(B):
            r = int(torch.randint(0, 8, (1,), generator=g))
            if r == 0:
                want.append(0)
            elif r == 1:
                want.append(max(0, lens[b] - 3))
            else:
                want.append(min(width * block, lens[b] + (T if T == 1 else int(torch.randint(1, T + 1, (1,), generator=g)))))
        q = torch.randn(B, Hq, 1, D, generator=g).to(dtype)
        kn, vn = (torch.randn(B, Hkv, T, D, generator=g).to(dtype) for _ in range(2))
        got = loop.step(torch.tensor(want, dtype=torch.int32, device=DEV), q.to(DEV), kn.to(DEV), vn.to(DEV)).cpu()
        ref, bound = loop.plain_step(want, q, kn, vn)
        assert loop.lens.tolist() == loop.p_lens and loop.state.tolist() == loop.p_state
        assert loop.table.tolist() == loop.p_table and loop.ring.tolist() == loop.p_ring
        assert bool(((got.double() - ref).abs() <= plain.tolerance(ref, bound, dtype)).all()), step


def test_two_captured_loops_replayed_together():
    """Two graphs of the whole step, captured on one stream and replayed side by side on two others,
    interleaved with eager calls, give what eager steps give."""
    B, Hq, Hkv, D, block, steps = 3, 8, 2, 128, 16, 6
    width, N = 64, 3 * 64
    g = _gen(23)
    prompt = [torch.randn(B, Hkv, 700, D, generator=g).bfloat16().to(DEV) for _ in range(4)]
    new = [[torch.randn(B, h, 1, D, generator=g).bfloat16().to(DEV) for h in (Hq, Hkv, Hkv)] for _ in range(steps)]
    q0 = torch.zeros(B, Hq, 1, D, dtype=torch.bfloat16, device=DEV)
    start = torch.tensor([700, 650, 333], dtype=torch.int32, device=DEV)
    loops = [_Loop(B, Hq, Hkv, D, block, width, N, torch.bfloat16) for _ in range(4)]
    for i, lp in enumerate(loops):
        lp.step(start, q0, prompt[i % 2 * 2], prompt[i % 2 * 2 + 1])
    want = [[], []]
    for i in (2, 3):  # eager
        for q, k, v in new:
            want[i - 2].append(loops[i].step(loops[i].lens + 1, q, k, v))
    graphs, ins, outs = [], [], []
    side = torch.cuda.Stream()
    for lp in loops[:2]:
        bufs = [t.clone() for t in new[0]]
        graph = torch.cuda.CUDAGraph()
        saved = [t.clone() for t in (lp.lens, lp.state)]
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            o = lp.step(lp.lens + 1, *bufs)
        assert torch.equal(lp.lens, saved[0]) and torch.equal(lp.state, saved[1])
        graphs.append(graph)
        ins.append(bufs)
        outs.append(o)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    noise = _simple_call(B=3, Hq=8, Hkv=1, D=128, lens=(3000, 100, 2500))
    quiet = dominus_ultra_decode_paged(*noise)
    got = [[], []]
    torch.cuda.synchronize()
    for s in range(steps):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                for dst, src in zip(ins[i], new[s]):
                    dst.copy_(src)
                graphs[i].replay()
                got[i].append(outs[i].clone())
        assert torch.equal(dominus_ultra_decode_paged(*noise), quiet)
    torch.cuda.synchronize()
    for i in (0, 1):
        for a, b in zip(got[i], want[i]):
            assert torch.equal(a, b)


def test_prompt_then_decode_agrees_with_prefill():
    """The attention of the last token of a prompt, from the cache, against the prefill's last row on
    the same values: keys and values whose 8-bit form is exact (small multiples of a power of two,
    unrotated positions apart), so only the kernels' own errors remain."""
    B, Hq, Hkv, T, D, block = 2, 8, 2, 200, 64, 32
    g = _gen(31)
    cos = torch.ones(T, D // 2, dtype=torch.bfloat16, device=DEV)
    sin = torch.zeros(T, D // 2, dtype=torch.bfloat16, device=DEV)
    k, v = ((torch.randint(-7, 8, (B, Hkv, T, D), generator=g).float() / 8).bfloat16().to(DEV) for _ in range(2))
    q = torch.randn(B, Hq, T, D, generator=g).bfloat16().to(DEV)
    full, _ = dominus_ultra_prefill(q, k, v, cos, sin, Hkv)
    lp = _Loop(B, Hq, Hkv, D, block, 8, 16, torch.bfloat16)
    lp.cos, lp.sin = cos, sin
    out = lp.step(torch.tensor([T, T], dtype=torch.int32, device=DEV), q[:, :, -1:].contiguous(), k, v)
    # each side: half a step of bf16 on its output, and the prefill's own gate for its bf16 weights
    assert (out.float() - full[:, :, -1:].float()).abs().max().item() <= 2e-2
