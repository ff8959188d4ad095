"""Host-side contract of the paged 8-bit cache (no GPU): refusals, host range checks, the C ABI's
argument checks, and the plain implementation's own properties."""

from __future__ import annotations

import ctypes

import pytest
import torch

import dominus_ultra
import dominusultra_b200
from dominusultra_b200 import (
    _lib,
    dominus_ultra_decode_paged,
    dominus_ultra_paged_tables,
    dominus_ultra_paged_write,
    paged,
    precompute_rope_cos_sin,
)
from tests import _paged as plain


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _cache(n=4, h=2, block=16, d=64):
    return torch.zeros(n, h, block, d, dtype=torch.uint8).view(torch.float8_e4m3fn)


def test_entry_points_are_exported():
    for name in paged.__all__:
        assert getattr(dominusultra_b200, name) is getattr(paged, name)
        assert getattr(dominus_ultra, name) is getattr(paged, name)


class TestTablesRefusals:
    def call(self, **kw):
        a = dict(block_table=_i32(2, 4), cache_seqlens=_i32(2), new_seqlens=_i32(2), free_blocks=_i32(8),
                 free_state=_i32(2), block_size=16, max_new=1)
        a.update(kw)
        return dominus_ultra_paged_tables(**a)

    @pytest.mark.parametrize("kw,match", [
        (dict(block_table=_i32(2)), "non-empty"),
        (dict(block_table=_i32(0, 4)), "non-empty"),
        (dict(block_size=24), "block_size"),
        (dict(block_size=8), "block_size"),
        (dict(max_new=-1), "max_new"),
        (dict(cache_seqlens=_i32(3)), r"cache_seqlens must have shape \[batch\]"),
        (dict(new_seqlens=torch.zeros(2)), "new_seqlens must be an int32 or int64"),
        (dict(free_blocks=_i32(0)), "free_blocks"),
        (dict(free_state=_i32(3)), "free_state"),
        (dict(), "require CUDA tensors"),
    ])
    def test_refused(self, kw, match):
        with pytest.raises(ValueError, match=match):
            self.call(**kw)


class TestWriteRefusals:
    def call(self, **kw):
        k = torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16)
        cos, sin = precompute_rope_cos_sin(8, 64, "cpu", torch.bfloat16)
        a = dict(k_new=k, v_new=k, k_cache=_cache(), v_cache=_cache(), k_scale=torch.zeros(4, 2),
                 v_scale=torch.zeros(4, 2), slots=_i32(2, 3), cache_seqlens=_i32(2), cos=cos, sin=sin)
        a.update(kw)
        return dominus_ultra_paged_write(**a)

    @pytest.mark.parametrize("kw,match", [
        (dict(k_new=torch.zeros(2, 3, 64)), "rank-4"),
        (dict(k_new=torch.zeros(2, 2, 0, 64), v_new=torch.zeros(2, 2, 0, 64)), "must be positive"),
        (dict(v_new=torch.zeros(2, 2, 4, 64)), "same shape"),
        (dict(k_cache=_cache(h=3)), "head count"),
        (dict(slots=_i32(2, 4)), "slots must have shape"),
        (dict(cache_seqlens=_i32(1)), "cache_seqlens must have shape"),
        (dict(), "require CUDA tensors"),
    ])
    def test_refused(self, kw, match):
        with pytest.raises(ValueError, match=match):
            self.call(**kw)


class TestDecodeRefusals:
    def call(self, **kw):
        cos, sin = precompute_rope_cos_sin(64, 64, "cpu", torch.bfloat16)
        a = dict(q_new=torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16), k_cache=_cache(), v_cache=_cache(),
                 k_scale=torch.ones(4, 2), v_scale=torch.ones(4, 2), block_table=_i32(2, 4),
                 cache_seqlens=_i32(2), cos=cos, sin=sin)
        a.update(kw)
        return dominus_ultra_decode_paged(**a)

    @pytest.mark.parametrize("kw,match", [
        (dict(q_new=torch.zeros(2, 4, 64)), "rank-4"),
        (dict(q_new=torch.zeros(2, 4, 2, 64)), "exactly one sequence position"),
        (dict(q_new=torch.zeros(0, 4, 1, 64)), "must be positive"),
        (dict(q_new=torch.zeros(2, 3, 1, 64)), "divisible"),
        (dict(k_cache=_cache(d=32)), "head_dim"),
        (dict(block_table=_i32(3, 4)), "block_table must have shape"),
        (dict(cache_seqlens=_i32(3)), "cache_seqlens must have shape"),
        (dict(q_new=torch.zeros(2, 4, 1, 48, dtype=torch.bfloat16), k_cache=_cache(d=48)), "power of two"),
        (dict(), "require CUDA tensors"),
    ])
    def test_refused(self, kw, match):
        with pytest.raises(ValueError, match=match):
            self.call(**kw)


class TestHostChecks:
    cpu = torch.device("cpu")

    def test_lengths(self):
        paged._check_host_lengths("cache_seqlens", torch.tensor([0, 5, 64]), 64)
        with pytest.raises(ValueError, match=r"cache_seqlens\[1\] = 65 is outside \[0, 64\]"):
            paged._check_host_lengths("cache_seqlens", torch.tensor([0, 65]), 64)
        with pytest.raises(ValueError, match=r"\[0\] = -1"):
            paged._check_host_lengths("new_seqlens", torch.tensor([-1, 0]), 64)

    def test_bad_pages(self):
        table = torch.tensor([[0, 3, -1], [2, 9, 99]], dtype=torch.int32)
        paged._check_host_table(table, torch.tensor([32, 16]), 16, 4)  # unused entries may hold anything
        with pytest.raises(ValueError, match=r"block_table\[0, 2\] = -1"):
            paged._check_host_table(table, torch.tensor([33, 16]), 16, 4)
        with pytest.raises(ValueError, match=r"block_table\[1, 1\] = 9"):
            paged._check_host_table(table, torch.tensor([32, 17]), 16, 4)

    def test_long_lengths_stay_out_of_range(self):
        got = paged._device_int32(torch.tensor([2**32 + 5, -(2**40), 7]), self.cpu)
        assert got.tolist() == [2**31 - 1, -1, 7] and got.dtype == torch.int32

    @pytest.mark.parametrize("change,match", [
        (dict(k_cache=_cache().float()), "float8_e4m3fn"),
        (dict(v_cache=_cache(n=5)), "same shape"),
        (dict(k_cache=_cache(block=24), v_cache=_cache(block=24)), "block_size"),
        (dict(k_scale=torch.ones(4, 3)), r"k_scale must have shape"),
        (dict(v_scale=torch.ones(4, 2).double()), "v_scale must use float32"),
        (dict(k_scale=torch.ones(2, 4).t()), "k_scale must be contiguous"),
        (dict(k_cache=_cache(h=4)[:, ::2]), "k_cache must be contiguous"),
    ])
    def test_cache(self, change, match):
        a = dict(k_cache=_cache(), v_cache=_cache(), k_scale=torch.ones(4, 2), v_scale=torch.ones(4, 2), device=self.cpu)
        paged._validate_paged_cache(**a)
        a.update(change)
        with pytest.raises(ValueError, match=match):
            paged._validate_paged_cache(**a)


def test_c_abi_rejects_bad_arguments():
    lib = _lib.load()
    null, fake, odd = ctypes.c_void_p(0), ctypes.c_void_p(0x10000), ctypes.c_void_p(0x10002)
    other = [ctypes.c_void_p(0x20000 + 0x1000 * i) for i in range(3)]

    def tables(**kw):
        a = dict(t=fake, o=fake, n=fake, r=fake, s=fake, sl=other[0], lo=other[1], so=other[2], B=2, w=4, N=8, bs=16, T=1)
        a.update(kw)
        return lib.du_paged_tables(*a.values(), null)

    assert tables(bs=48) == _lib.DU_ERR_UNSUPPORTED and "block_size" in _lib.last_error()
    assert tables(B=0) == _lib.DU_ERR_INVALID
    assert tables(B=8193) == _lib.DU_ERR_UNSUPPORTED and "8192" in _lib.last_error()
    assert tables(w=2**27, bs=16) == _lib.DU_ERR_UNSUPPORTED
    assert tables(N=2**27, bs=16) == _lib.DU_ERR_UNSUPPORTED and "2^31" in _lib.last_error()
    assert tables(sl=null) == _lib.DU_ERR_INVALID and "null" in _lib.last_error()
    assert tables(r=odd) == _lib.DU_ERR_INVALID and "4-byte" in _lib.last_error()
    assert tables(lo=fake) == _lib.DU_ERR_INVALID and "must not be the inputs" in _lib.last_error()

    def write(**kw):
        a = dict(k=fake, v=fake, kc=fake, vc=fake, ks=fake, vs=fake, sl=fake, pl=fake, c=fake, s=fake, B=1, H=2, T=3,
                 D=64, N=8, bs=16, dt=_lib.DU_DTYPE_BF16, rp=64)
        a.update(kw)
        return lib.du_paged_write(*a.values(), null)

    assert write(T=0) == _lib.DU_ERR_INVALID
    assert write(D=48) == _lib.DU_ERR_UNSUPPORTED
    assert write(dt=_lib.DU_DTYPE_F32) == _lib.DU_ERR_INVALID
    assert write(kc=odd) == _lib.DU_ERR_INVALID and "16-byte" in _lib.last_error()
    assert write(rp=0) == _lib.DU_ERR_INVALID

    def decode(**kw):
        a = dict(q=fake, kc=fake, vc=fake, ks=fake, vs=fake, t=fake, ln=fake, c=fake, s=fake, o=fake, B=1, Hq=4, Hkv=2,
                 D=64, N=8, bs=16, w=4, dt=_lib.DU_DTYPE_BF16, sc=0.125, rp=64, tk=fake, ws=fake, wsb=1 << 30)
        a.update(kw)
        return lib.du_decode_paged(*a.values(), null)

    assert decode(Hq=3) == _lib.DU_ERR_INVALID and "divisible" in _lib.last_error()
    assert decode(w=0) == _lib.DU_ERR_INVALID
    assert decode(bs=256) == _lib.DU_ERR_UNSUPPORTED
    assert decode(t=odd) == _lib.DU_ERR_INVALID and "4-byte" in _lib.last_error()
    assert decode(o=null) == _lib.DU_ERR_INVALID
    assert decode(D=512) == _lib.DU_ERR_UNSUPPORTED
    assert decode(tk=null) == _lib.DU_ERR_INVALID
    assert decode(wsb=0) == _lib.DU_ERR_WORKSPACE and decode(ws=null) == _lib.DU_ERR_WORKSPACE
    assert decode(sc=0.0) == _lib.DU_ERR_INVALID
    assert lib.du_decode_paged_workspace_size(1, 4, 2, 64, 16, 4) > 0
    assert lib.du_decode_paged_workspace_size(1, 3, 2, 64, 16, 4) == 0


class TestPlain:
    def test_units(self):
        assert plain.unit_of(448.0) == 1.0 and plain.unit_of(448.001) == 2.0 and plain.unit_of(224.0) == 0.5
        assert plain.unit_of(0.0) == 2.0**-64

    def test_nearest_agrees_with_torch(self):
        g = torch.Generator().manual_seed(3)
        x = torch.randn(20000, generator=g) * 30
        x = x.clamp(-448, 448)
        assert torch.equal(plain.nearest_e4m3(x.double()), x.to(torch.float8_e4m3fn).double())

    def test_ring_conserves_blocks(self):
        g = torch.Generator().manual_seed(5)
        block, width, B, N = 16, 6, 5, 24
        table = [[-1] * width for _ in range(B)]
        ring, state, lens = list(range(N)), [0, N], [0] * B
        for _ in range(200):
            want = torch.randint(0, width * block + 1, (B,), generator=g).tolist()
            want = [min(w, n + 20) for w, n in zip(want, lens)]
            _, lens, state = plain.tables(table, lens, want, ring, state, block, 20)
            held = [table[b][i] for b in range(B) for i in range(plain.pages(lens[b], block))]
            free = [ring[(state[0] + i) % N] for i in range(state[1])]
            assert sorted(held + free) == list(range(N))
