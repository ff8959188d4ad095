"""What the paged entry points refuse of tensors on the GPU: every argument with a wrong type, shape, stride,
device or alignment is refused by name and nothing is written; what is allowed beside that is taken."""

from __future__ import annotations

import pytest
import torch

from dominusultra_b200 import (
    _lib,
    dominus_ultra_decode_paged,
    dominus_ultra_paged_tables,
    dominus_ultra_paged_write,
    precompute_rope_cos_sin,
)

pytestmark = pytest.mark.gpu

DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)
B, HQ, HKV, D, BLOCK, N, T, WIDTH = 2, 4, 2, 64, 16, 8, 3, 4


@pytest.fixture(autouse=True)
def _clean_status(cuda_device):
    _lib.read_status(reset=True)
    yield
    assert _lib.read_status(reset=True)[0] == 0, "a test left a device status"


def _strided(t):
    """The same values with gaps between the elements of the last dimension."""
    wide = torch.zeros(*t.shape, 2, dtype=t.dtype, device=t.device)
    view = wide[..., 0]
    view.copy_(t)
    assert not view.is_contiguous()
    return view


def _shifted(t, by=1):
    """The same values at an address that is not a multiple of 16 bytes."""
    flat = torch.zeros(t.numel() + by, dtype=t.dtype, device=t.device)[by:]
    view = flat.view(t.shape)
    view.view(torch.uint8 if t.element_size() == 1 else t.dtype).copy_(t.view(torch.uint8) if t.element_size() == 1 else t)
    assert view.is_contiguous() and view.data_ptr() % 16
    return view


def _cache(g, shape=(N, HKV, BLOCK, D)):
    return torch.randn(*shape, generator=g, device=DEV).to(torch.float8_e4m3fn)


def _tables():
    return dict(block_table=torch.tensor([[0, -1, -1, -1], [1, 2, -1, -1]], **I32), cache_seqlens=torch.tensor([5, 20], **I32),
                new_seqlens=torch.tensor([8, 21], **I32), free_blocks=torch.tensor([3, 4, 5, 6, 7, -1, -1, -1], **I32),
                free_state=torch.tensor([0, 5], **I32), block_size=BLOCK, max_new=T)


def _write():
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn(B, HKV, T, D, generator=g, device=DEV).bfloat16() for _ in range(2))
    cos, sin = precompute_rope_cos_sin(64, D, DEV, torch.bfloat16)
    return dict(k_new=k, v_new=v, k_cache=_cache(g), v_cache=_cache(g), k_scale=torch.ones(N, HKV, device=DEV),
                v_scale=torch.ones(N, HKV, device=DEV), slots=torch.tensor([[5, 6, 7], [36, 37, -1]], **I32),
                cache_seqlens=torch.tensor([5, 20], **I32), cos=cos, sin=sin)


def _decode():
    g = torch.Generator(device=DEV).manual_seed(2)
    cos, sin = precompute_rope_cos_sin(64, D, DEV, torch.bfloat16)
    return dict(q_new=torch.randn(B, HQ, 1, D, generator=g, device=DEV).bfloat16(), k_cache=_cache(g), v_cache=_cache(g),
                k_scale=torch.ones(N, HKV, device=DEV), v_scale=torch.ones(N, HKV, device=DEV),
                block_table=torch.tensor([[0, -1, -1, -1], [1, 2, 3, -1]], **I32), cache_seqlens=torch.tensor([5, 40], **I32),
                cos=cos, sin=sin)


MAKE = {"tables": (_tables, dominus_ultra_paged_tables), "write": (_write, dominus_ultra_paged_write), "decode": (_decode, dominus_ultra_decode_paged)}
CPU = lambda t: t.cpu()  # noqa: E731
LONG = lambda t: t.long()  # noqa: E731

TABLES = [
    ("block_table", LONG, "block_table must be an int32"),
    ("block_table", _strided, "block_table must be contiguous"),
    ("block_table", lambda t: t[0], "non-empty"),
    ("block_table", lambda t: t[:, :0], "non-empty"),
    ("block_table", CPU, "require CUDA tensors"),
    ("cache_seqlens", lambda t: t.float(), "cache_seqlens must be an int32 or int64"),
    ("cache_seqlens", lambda t: t[:1], r"cache_seqlens must have shape \[batch\]"),
    ("cache_seqlens", lambda t: t[None], r"cache_seqlens must have shape \[batch\]"),
    ("cache_seqlens", lambda t: t.cpu() + 100, r"cache_seqlens\[0\] = 105 is outside"),
    ("new_seqlens", lambda t: t.bool(), "new_seqlens must be an int32 or int64"),
    ("new_seqlens", lambda t: torch.cat([t, t]), r"new_seqlens must have shape \[batch\]"),
    ("new_seqlens", lambda t: t.cpu() - 9, r"new_seqlens\[0\] = -1 is outside"),
    ("free_blocks", LONG, "free_blocks must be an int32"),
    ("free_blocks", _strided, "free_blocks must be contiguous"),
    ("free_blocks", lambda t: t[None], "free_blocks must be a non-empty"),
    ("free_blocks", lambda t: t[:0], "free_blocks must be a non-empty"),
    ("free_blocks", CPU, "free_blocks must be on the same"),
    ("free_state", LONG, "free_state must be an int32"),
    ("free_state", lambda t: torch.cat([t, t]), "free_state must have shape"),
    ("free_state", _strided, "free_state must be contiguous"),
    ("free_state", CPU, "free_state must be on the same"),
    ("block_size", lambda _: 24, "block_size must be"),
    ("block_size", lambda _: 256, "block_size must be"),
    ("max_new", lambda _: -1, "max_new must not be negative"),
]
CACHES = [
    ("k_cache", lambda t: t.view(torch.uint8), "k_cache must use float8_e4m3fn"),
    ("v_cache", lambda t: t.view(torch.uint8).view(torch.float8_e5m2), "v_cache must use float8_e4m3fn"),
    ("k_cache", lambda t: t.view(torch.uint8).transpose(0, 1).contiguous().transpose(0, 1).view(torch.float8_e4m3fn), "k_cache must be contiguous"),
    ("v_cache", lambda t: t.view(torch.uint8).transpose(0, 1).contiguous().transpose(0, 1).view(torch.float8_e4m3fn), "v_cache must be contiguous"),
    ("k_cache", lambda t: _shifted(t, 8), "k_cache must be 16-byte aligned"),
    ("v_cache", lambda t: _shifted(t, 4), "v_cache must be 16-byte aligned"),
    ("k_cache", CPU, "same CUDA device"),
    ("v_cache", CPU, "same CUDA device"),
    ("v_cache", lambda t: t[:-1], "same shape"),
    ("v_cache", lambda t: t[0], "rank-4"),
    ("k_scale", lambda t: t.double(), "k_scale must use float32"),
    ("v_scale", lambda t: t.half(), "v_scale must use float32"),
    ("k_scale", lambda t: t.t(), "k_scale must have shape"),
    ("v_scale", lambda t: t[:, :1], "v_scale must have shape"),
    ("k_scale", _strided, "k_scale must be contiguous"),
    ("v_scale", _strided, "v_scale must be contiguous"),
    ("k_scale", CPU, "same CUDA device"),
    ("v_scale", CPU, "same CUDA device"),
]
ROPE = [
    ("cos", lambda t: t.float(), "same dtype"),
    ("sin", lambda t: t.half(), "same dtype"),
    ("cos", _strided, "contiguous"),
    ("sin", _strided, "contiguous"),
    ("cos", CPU, "same device"),
    ("sin", CPU, "same device"),
    ("cos", lambda t: t[:, :16].contiguous(), "trailing shape"),
    ("sin", lambda t: torch.cat([t, t], 1), "trailing shape"),
    ("cos", lambda t: t[0], "rank-2"),
    ("sin", lambda t: t[:0], "at least 1"),
]
WRITE = CACHES + ROPE + [
    ("k_new", lambda t: t.float(), "float16 or bfloat16"),
    ("v_new", lambda t: t.half(), "same dtype"),
    ("k_new", lambda t: t.transpose(1, 2).contiguous().transpose(1, 2), "must be contiguous"),
    ("v_new", _strided, "must be contiguous"),
    ("k_new", CPU, "require CUDA tensors"),
    ("v_new", CPU, "same CUDA device"),
    ("v_new", lambda t: t[:, :, :2].contiguous(), "same shape"),
    ("k_new", lambda t: t[0], "rank-4"),
    ("slots", LONG, "slots must be an int32"),
    ("slots", _strided, "slots must be contiguous"),
    ("slots", CPU, "slots must be on the same"),
    ("slots", lambda t: t[:, :2].contiguous(), "slots must have shape"),
    ("cache_seqlens", lambda t: t.float(), "cache_seqlens must be an int32 or int64"),
    ("cache_seqlens", lambda t: t[:1], "cache_seqlens must have shape"),
    ("cache_seqlens", lambda t: t.cpu() + 60, r"cache_seqlens\[0\] = 65 is outside"),
]
DECODE = CACHES + ROPE + [
    ("q_new", lambda t: t.float(), "float16 or bfloat16"),
    ("q_new", lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), "must be contiguous"),
    ("q_new", CPU, "require CUDA tensors"),
    ("q_new", lambda t: t[0], "rank-4"),
    ("q_new", lambda t: torch.cat([t, t], 2), "exactly one sequence position"),
    ("q_new", lambda t: t[:, :3].contiguous(), "divisible"),
    ("q_new", lambda t: t[..., :32].contiguous(), "head_dim"),
    ("block_table", LONG, "block_table must be an int32"),
    ("block_table", _strided, "block_table must be contiguous"),
    ("block_table", lambda t: t[:1], "block_table must have shape"),
    ("block_table", lambda t: t[:, :0], "block_table must have shape"),
    ("cache_seqlens", lambda t: t.float(), "cache_seqlens must be an int32 or int64"),
    ("cache_seqlens", lambda t: t[None], "cache_seqlens must have shape"),
    ("cache_seqlens", lambda t: t.cpu() + 30, r"cache_seqlens\[1\] = 70 is outside"),
]
ALL = [("tables", *x) for x in TABLES] + [("write", *x) for x in WRITE] + [("decode", *x) for x in DECODE]


def _bits(t):
    return t.contiguous().view(torch.uint8) if t.element_size() == 1 else t


@pytest.mark.parametrize("op,name,change,match", ALL, ids=[f"{o}-{n}-{i}" for i, (o, n, *_) in enumerate(ALL)])
def test_refused(op, name, change, match):
    make, call = MAKE[op]
    args = make()
    args[name] = change(args[name])
    before = {k: v.clone() for k, v in args.items() if torch.is_tensor(v)}
    with pytest.raises(ValueError, match=match):
        call(**args)
    for k, v in before.items():
        assert torch.equal(_bits(args[k]), _bits(v)), k


@pytest.mark.parametrize("op", MAKE)
def test_the_unchanged_call_is_taken(op):
    make, call = MAKE[op]
    call(**make())


# What is taken beside the exact form: lengths of 64 bits, on the host or with gaps, inputs at any address.
TAKEN = [("tables", n, c) for n in ("cache_seqlens", "new_seqlens") for c in (LONG, CPU, _strided)]
TAKEN += [("write", "cache_seqlens", c) for c in (LONG, CPU, _strided)] + [("decode", "cache_seqlens", c) for c in (LONG, CPU, _strided)]
TAKEN += [("write", n, _shifted) for n in ("k_new", "v_new", "cos", "sin")] + [("decode", n, _shifted) for n in ("q_new", "cos", "sin")]
TAKEN += [("decode", "block_table", CPU)]


@pytest.mark.parametrize("op,name,change", TAKEN, ids=[f"{o}-{n}-{i}" for i, (o, n, _) in enumerate(TAKEN)])
def test_taken(op, name, change):
    make, call = MAKE[op]
    plain, args = make(), make()
    args[name] = change(args[name])
    if op == "decode" and name == "block_table":
        plain["cache_seqlens"] = plain["cache_seqlens"].cpu()
        args["cache_seqlens"] = args["cache_seqlens"].cpu()
    want, got = call(**plain), call(**args)
    for a, b in zip(got if op == "tables" else [got] if op == "decode" else [], want if op == "tables" else [want] if op == "decode" else []):
        assert torch.equal(a, b)
    for k in ("block_table", "free_blocks", "k_cache", "v_cache", "k_scale", "v_scale"):
        if k in args:
            assert torch.equal(_bits(args[k].cuda()), _bits(plain[k].cuda())), k
