"""Forks, copies, compactions and the attention of several new tokens without a GPU: refusals of the
Python and C entry points, and properties of the plain implementations that the GPU tests use."""

from __future__ import annotations

import ctypes

import pytest
import torch

import dominus_ultra
import dominusultra_b200 as du
from dominusultra_b200 import _lib
from tests import _paged_shared as plain

NAMES = ["dominus_ultra_extend_paged", "dominus_ultra_paged_fork", "dominus_ultra_paged_copy", "dominus_ultra_paged_compact"]


@pytest.mark.parametrize("name", NAMES)
def test_exported(name):
    assert getattr(du, name) is getattr(dominus_ultra, name)


def _ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def _fork(**kw):
    a = dict(block_table=_ints(2, 3), cache_seqlens=_ints(2), sources=_ints(2), new_seqlens=_ints(2), free_blocks=_ints(8), free_state=_ints(2), block_size=16)
    a.update(kw)
    return du.dominus_ultra_paged_fork(**a)


def _compact(**kw):
    a = dict(block_table=_ints(2, 3), cache_seqlens=_ints(2), free_blocks=_ints(8), free_state=_ints(2), block_size=16)
    a.update(kw)
    return du.dominus_ultra_paged_compact(**a)


@pytest.mark.parametrize("call", [_fork, _compact])
@pytest.mark.parametrize(
    "kw,message",
    [
        (dict(block_table=_ints(2)), "non-empty"),
        (dict(block_table=_ints(0, 3), cache_seqlens=_ints(0)), "non-empty"),
        (dict(block_size=48), "block_size"),
        (dict(cache_seqlens=_ints(3)), "cache_seqlens must have shape"),
        (dict(cache_seqlens=_ints(2).float()), "cache_seqlens must be an int32 or int64"),
        (dict(free_blocks=_ints(0)), "free_blocks"),
        (dict(free_blocks=_ints(2, 4)), "free_blocks"),
        (dict(free_state=_ints(3)), "free_state"),
        (dict(), "require CUDA"),
    ],
)
def test_refusals_of_tables(call, kw, message):
    with pytest.raises(ValueError, match=message):
        call(**kw)


@pytest.mark.parametrize("kw,message", [(dict(sources=_ints(3)), "sources must have shape"), (dict(new_seqlens=_ints(2, 1)), "new_seqlens must have shape"), (dict(sources=_ints(2).float()), "sources must be")])
def test_refusals_of_a_fork(kw, message):
    with pytest.raises(ValueError, match=message):
        _fork(**kw)


def _cache(N=4, H=2, block=16, D=64):
    return torch.zeros(N, H, block, D).to(torch.float8_e4m3fn), torch.ones(N, H)


@pytest.mark.parametrize(
    "kw,message",
    [
        (dict(k_cache=torch.zeros(4, 2, 16)), "rank-4"),
        (dict(copies=_ints(4)), "copies must have shape"),
        (dict(copies=_ints(4, 3)), "copies must have shape"),
        (dict(k_cache=_cache(D=48)[0]), "head_dim"),
        (dict(), "require CUDA"),
    ],
)
def test_refusals_of_a_copy(kw, message):
    k, s = _cache()
    a = dict(k_cache=k, v_cache=k, k_scale=s, v_scale=s, copies=_ints(3, 2))
    a.update(kw)
    with pytest.raises(ValueError, match=message):
        du.dominus_ultra_paged_copy(**a)


@pytest.mark.parametrize(
    "kw,message",
    [
        (dict(q_new=torch.zeros(2, 4, 64)), "rank-4"),
        (dict(q_new=torch.zeros(2, 4, 0, 64).bfloat16()), "must be positive"),
        (dict(q_new=torch.zeros(2, 3, 5, 64).bfloat16()), "divisible"),
        (dict(q_new=torch.zeros(2, 4, 5, 32).bfloat16()), "head_dim"),
        (dict(block_table=_ints(3, 4)), "block_table"),
        (dict(block_table=_ints(2, 0)), "block_table"),
        (dict(past_seqlens=_ints(3)), "past_seqlens must have shape"),
        (dict(cache_seqlens=_ints(2).float()), "cache_seqlens must be"),
        (dict(), "require CUDA"),
    ],
)
def test_refusals_of_an_extension(kw, message):
    k, s = _cache()
    t = torch.ones(64, 32).bfloat16()
    a = dict(q_new=torch.zeros(2, 4, 5, 64).bfloat16(), k_cache=k, v_cache=k, k_scale=s, v_scale=s, block_table=_ints(2, 4), past_seqlens=_ints(2), cache_seqlens=_ints(2), cos=t, sin=t)
    a.update(kw)
    with pytest.raises(ValueError, match=message):
        du.dominus_ultra_extend_paged(**a)


def test_c_entry_points_refuse():
    lib = _lib.load()
    null, fake, odd = ctypes.c_void_p(0), ctypes.c_void_p(0x10000), ctypes.c_void_p(0x10002)
    other = [ctypes.c_void_p(0x20000 + 0x1000 * i) for i in range(4)]

    def fork(**kw):
        a = dict(t=fake, ln=fake, s=fake, w=fake, r=fake, st=fake, to=other[0], c=other[1], lo=other[2], so=other[3], B=2, width=4, N=8, bs=16)
        a.update(kw)
        return lib.du_paged_fork(*a.values(), null)

    def compact(**kw):
        a = dict(t=fake, ln=fake, r=fake, st=fake, to=other[0], c=other[1], ro=other[2], so=other[3], B=2, width=4, N=8, bs=16, ws=fake, wsb=1 << 20)
        a.update(kw)
        return lib.du_paged_compact(*a.values(), null)

    for call in (fork, compact):
        assert call(bs=8) == _lib.DU_ERR_UNSUPPORTED and "block_size" in _lib.last_error()
        assert call(B=0) == _lib.DU_ERR_INVALID
        assert call(B=8193) == _lib.DU_ERR_UNSUPPORTED and "8192" in _lib.last_error()
        assert call(N=0) == _lib.DU_ERR_INVALID
        assert call(N=2**20) == _lib.DU_ERR_UNSUPPORTED and "shared memory" in _lib.last_error()
        assert call(width=2**27) == _lib.DU_ERR_UNSUPPORTED
        assert call(t=null) == _lib.DU_ERR_INVALID and "null" in _lib.last_error()
        assert call(to=null) == _lib.DU_ERR_INVALID
        assert call(ln=odd) == _lib.DU_ERR_INVALID and "4-byte" in _lib.last_error()
        assert call(so=odd) == _lib.DU_ERR_INVALID and "4-byte" in _lib.last_error()
        assert call(to=fake) == _lib.DU_ERR_INVALID and "must not be the inputs" in _lib.last_error()
    assert compact(ws=null) == _lib.DU_ERR_WORKSPACE and compact(wsb=31) == _lib.DU_ERR_WORKSPACE
    assert compact(ws=ctypes.c_void_p(0x10008)) == _lib.DU_ERR_INVALID and "workspace" in _lib.last_error()
    assert fork(N=2**19) == _lib.DU_ERR_UNSUPPORTED and "shared memory" in _lib.last_error()
    assert fork(N=250000, B=8192) == _lib.DU_ERR_UNSUPPORTED and "shared memory" in _lib.last_error()
    # (what the Python call passes)
    assert all(lib.du_paged_compact_workspace_size(n) == 16 * (1 + (n + 127) // 128 * 4) for n in (1, 128, 129, 770000))
    assert lib.du_paged_compact_workspace_size(0) == lib.du_paged_compact_workspace_size(770001) == 0

    def copy(**kw):
        a = dict(k=fake, v=fake, ks=fake, vs=fake, c=fake, n=3, N=8, H=2, bs=16, D=64)
        a.update(kw)
        return lib.du_paged_copy(*a.values(), null)

    assert copy(n=-1) == _lib.DU_ERR_INVALID
    assert copy(n=0) == _lib.DU_OK
    assert copy(D=24) == _lib.DU_ERR_UNSUPPORTED
    assert copy(H=0) == _lib.DU_ERR_INVALID
    assert copy(c=null) == _lib.DU_ERR_INVALID
    assert copy(v=ctypes.c_void_p(0x10004)) == _lib.DU_ERR_INVALID and "16-byte" in _lib.last_error()
    assert copy(c=odd) == _lib.DU_ERR_INVALID and "4-byte" in _lib.last_error()

    def extend(**kw):
        a = dict(q=fake, kc=fake, vc=fake, ks=fake, vs=fake, t=fake, p=fake, ln=fake, c=fake, s=fake, o=fake, B=1, Hq=4, Hkv=2, T=3,
                 D=64, N=8, bs=16, w=4, dt=_lib.DU_DTYPE_BF16, sc=0.125, rp=64, ws=fake, wsb=1 << 32)
        a.update(kw)
        return lib.du_extend_paged(*a.values(), null)

    assert extend(Hq=3) == _lib.DU_ERR_INVALID and "divisible" in _lib.last_error()
    assert extend(T=0) == _lib.DU_ERR_INVALID
    assert extend(D=512) == _lib.DU_ERR_UNSUPPORTED
    assert extend(bs=256) == _lib.DU_ERR_UNSUPPORTED
    assert extend(w=0) == _lib.DU_ERR_INVALID
    assert extend(w=2**24) == _lib.DU_ERR_UNSUPPORTED
    assert extend(p=null) == _lib.DU_ERR_INVALID
    assert extend(q=odd) == _lib.DU_ERR_INVALID and "16-byte" in _lib.last_error()
    assert extend(p=odd) == _lib.DU_ERR_INVALID and "4-byte" in _lib.last_error()
    assert extend(rp=0) == _lib.DU_ERR_INVALID
    assert extend(sc=0.0) == _lib.DU_ERR_INVALID
    assert extend(dt=_lib.DU_DTYPE_F32) == _lib.DU_ERR_INVALID
    assert extend(wsb=0) == _lib.DU_ERR_WORKSPACE and extend(ws=null) == _lib.DU_ERR_WORKSPACE
    assert lib.du_extend_paged_workspace_size(1, 4, 2, 3, 64, 16, 4) > 0
    assert lib.du_extend_paged_workspace_size(1, 3, 2, 3, 64, 16, 4) == 0


class TestPlain:
    def test_forks_conserve_blocks(self):
        g = torch.Generator().manual_seed(2)
        block, width, B, N = 16, 5, 6, 40
        table, lens = [[-1] * width for _ in range(B)], [0] * B
        table[0], lens[0] = list(range(5)), 77
        ring, state = list(range(5, N)) + [-1] * 5, [0, N - 5]
        for _ in range(300):
            s = torch.randint(0, B, (B,), generator=g).tolist()
            w = [int(torch.randint(0, lens[x] + 1, (1,), generator=g)) if int(torch.randint(0, 4, (1,), generator=g)) == 0 else lens[x] for x in s]
            if not any(lens):
                break
            table, copies, lens, state = plain.fork(table, lens, s, w, ring, state, block)
            held = [table[b][: plain.pages(n, block)] for b, n in enumerate(lens)]
            used = {x for r in held for x in r}
            free = [ring[(state[0] + i) % N] for i in range(state[1])]
            assert sorted(list(used) + free) == list(range(N))
            # a block that will be written is held by one request only
            for b, (r, n) in enumerate(zip(held, lens)):
                if n % block:
                    assert sum(r[-1] in x for x in held) == 1
            assert not {c[0] for c in copies if c[0] >= 0} & {c[1] for c in copies if c[0] >= 0}

    def test_compactions_keep_what_rows_hold(self):
        g = torch.Generator().manual_seed(3)
        for _ in range(50):
            N = int(torch.randint(1, 60, (1,), generator=g))
            order = torch.randperm(N, generator=g).tolist()
            held = order[: N // 2]
            table = [held[:5] + [-1] * (30 - len(held[:5])), held + [-1] * (30 - len(held))]
            lens = [16 * len(held[:5]), 16 * len(held)]
            free = order[N // 2 : N // 2 + N // 3]
            ring = free + [-1] * (N - len(free))
            out, moves, left, state = plain.compact(table, lens, ring, [0, len(free)], 16)
            content = list(range(N))
            for a, b in moves:
                if a >= 0:
                    content[b] = content[a]
            assert [content[x] for x in out[1][: len(held)]] == held and [content[x] for x in out[0][: len(held[:5])]] == held[:5]
            assert sorted(left[: state[1]] + out[1][: len(held)]) == sorted(free + held)
            assert not held or not free or max(out[1][: len(held)]) < min(left[: state[1]])
