"""Attention of several new tokens per request over the paged 8-bit cache.

``dominus_ultra_decode_paged`` answers one token per request. A prompt that is cached in chunks, a
question behind a long text, or a draft of several tokens asks for more: their keys and values are
written first (``dominus_ultra_paged_write``), then ``dominus_ultra_extend_paged`` attends to them and to
what was cached before (the causal rows of ``dominus_ultra_prefill``, reference
``dominus_ultra.py:416-501``, that lie behind ``past_seqlens[b]``).
"""

from __future__ import annotations

import torch

from . import _lib
from .attention import _aligned, _OnDevice, _validate_attention_tensors, _validate_head_dim
from .paged import (
    _CODES,
    _GET_DEVICE,
    _HEAD_DIMS,
    _check_host_lengths,
    _check_host_table,
    _device_int32,
    _fit_cache,
    _fit_rope,
    _lengths,
    _stream_of,
    _validate_int32,
    _validate_paged_cache,
    _workspace,
    _validate_tables_like,
)

__all__ = ["dominus_ultra_extend_paged"]

_I32 = torch.int32
# Sizes by what they depend on (head_dim, and whether the new tokens' rows of a KV head fill a row tile), so that a
# server whose batches, chunks and tables vary keeps no more than a few.
_WS_SIZES = {}


def _workspace_size(B, Hq, Hkv, T, D, block_size, max_blocks, index) -> int:
    key = (D, T * (Hq // Hkv) > 128, index)
    n = _WS_SIZES.get(key)
    if n is None:
        n = int(_lib.load().du_extend_paged_workspace_size(B, Hq, Hkv, T, D, block_size, max_blocks))
        if n:  # (0: sizes that the call will refuse)
            _WS_SIZES[key] = n
    return n


def dominus_ultra_extend_paged(
    q_new: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_table: torch.Tensor,
    past_seqlens: torch.Tensor,
    cache_seqlens: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
) -> torch.Tensor:
    """
    Attention of new tokens over the paged 8-bit cache that they extend (``du_extend_paged``).

    Request ``b`` had ``past_seqlens[b]`` tokens cached (what ``dominus_ultra_paged_tables`` and
    ``dominus_ultra_paged_write`` took) and has ``cache_seqlens[b]`` with its new ones (what the tables
    returned). Its new token ``t`` rotates at position ``past_seqlens[b] + t`` and attends to the keys
    up to its own. Rows behind a request's last new token are zeros. Rows of a block behind the length are
    never used, whatever they hold.

    Query rows and softmax weights are carried as fp16, as in ``dominus_ultra_prefill``. On unit-normal queries fp16
    outputs are off by about 0.0005 of their norm, 2.5 times what their own rounding takes (and
    ``dominus_ultra_decode_paged`` with it); bf16 outputs by no more than their own rounding.

    Lengths and table are read on the GPU: lengths out of range give zeros, a block id out of range
    NaN in the rows that see its keys, and ``_lib.read_status()`` reports code 6 or 7. Given on the CPU,
    they are checked here (a table only if ``cache_seqlens`` is there too).

    Args:
        q_new: [batch, num_heads, T, head_dim], not rotated
        k_cache, v_cache: [num_blocks, num_kv_heads, block_size, head_dim] float8_e4m3fn
        k_scale, v_scale: [num_blocks, num_kv_heads] fp32, positive
        block_table: [batch, max_blocks] int32
        past_seqlens: [batch] integer lengths before the new tokens
        cache_seqlens: [batch] integer lengths with them, at most T more
        cos, sin: tables from precompute_rope_cos_sin covering every length

    Returns:
        Output tensor of shape [batch, num_heads, T, head_dim]
    """
    shape, cache, table = q_new.shape, k_cache.shape, block_table.shape
    index, dtype = q_new.get_device(), q_new.dtype
    if not (
        len(shape) == 4 and len(cache) == 4 and len(table) == 2 and index >= 0 and dtype in _CODES
        and q_new.is_contiguous() and _fit_rope(cos, sin, dtype, index, shape[3])
        and shape[0] > 0 and shape[1] > 0 and shape[2] > 0 and shape[3] in _HEAD_DIMS
        and _fit_cache(k_cache, v_cache, k_scale, v_scale, cache, index)
        and shape[1] % cache[1] == 0 and cache[3] == shape[3]
        and block_table.dtype is _I32 and block_table.get_device() == index and block_table.is_contiguous()
        and table[0] == shape[0] and table[1] > 0
        and past_seqlens.dtype is _I32 and past_seqlens.get_device() == index and past_seqlens.is_contiguous()
        and cache_seqlens.dtype is _I32 and cache_seqlens.get_device() == index and cache_seqlens.is_contiguous()
        and past_seqlens.dim() == 1 and past_seqlens.shape[0] == shape[0]
        and cache_seqlens.dim() == 1 and cache_seqlens.shape[0] == shape[0]
    ):
        block_table, past_seqlens, cache_seqlens = _check_extend(
            q_new, k_cache, v_cache, k_scale, v_scale, block_table, past_seqlens, cache_seqlens, cos, sin
        )
    if _GET_DEVICE() != index:
        with _OnDevice(q_new.device):
            return dominus_ultra_extend_paged(
                q_new, k_cache, v_cache, k_scale, v_scale, block_table, past_seqlens, cache_seqlens, cos, sin
            )
    B, Hq, T, D = shape
    num_blocks, Hkv, block_size, _ = cache
    max_blocks = table[1]
    q, c, s = q_new.data_ptr(), cos.data_ptr(), sin.data_ptr()
    if (q | c | s) & 15:
        q_new, cos, sin = (_aligned(t) for t in (q_new, cos, sin))
        q, c, s = q_new.data_ptr(), cos.data_ptr(), sin.data_ptr()
    out = torch.empty_like(q_new)
    stream = _stream_of(index)
    nbytes = _workspace_size(B, Hq, Hkv, T, D, block_size, max_blocks, index)
    ws, keep = _workspace(nbytes, index, stream)
    rc = _lib.load().du_extend_paged(
        q, k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), block_table.data_ptr(),
        past_seqlens.data_ptr(), cache_seqlens.data_ptr(), c, s, out.data_ptr(), B, Hq, Hkv, T, D, num_blocks,
        block_size, max_blocks, _CODES[dtype], D**-0.5, min(cos.shape[0], sin.shape[0]), ws, nbytes, stream,
    )
    del keep
    if rc:
        _lib.check(rc, "du_extend_paged")
    return out


def _check_extend(q_new, k_cache, v_cache, k_scale, v_scale, block_table, past_seqlens, cache_seqlens, cos, sin):
    """The refusals of dominus_ultra_extend_paged; returns the table and the lengths on the device."""
    if q_new.ndim != 4 or k_cache.ndim != 4 or v_cache.ndim != 4:
        raise ValueError("q_new, k_cache, and v_cache must be rank-4 tensors")
    B, Hq, T, D = q_new.shape
    if B <= 0 or Hq <= 0 or T <= 0:
        raise ValueError("batch, heads, and sequence length must be positive")
    Hkv = k_cache.shape[1]
    if Hkv <= 0 or Hq % Hkv != 0:
        raise ValueError("num_query_heads must be divisible by num_kv_heads")
    if k_cache.shape[3] != D:
        raise ValueError("the caches must have q_new's head_dim")
    if block_table.ndim != 2 or block_table.shape[0] != B or block_table.shape[1] <= 0:
        raise ValueError("block_table must have shape [batch, max_blocks]")
    _lengths("past_seqlens", past_seqlens, B)
    _lengths("cache_seqlens", cache_seqlens, B)
    _validate_head_dim(D)
    _validate_attention_tensors(q_new)
    device = q_new.device
    _validate_paged_cache(k_cache, v_cache, k_scale, v_scale, device)
    _validate_tables_like(cos, sin, D, device, q_new.dtype)
    num_blocks, _, block_size, _ = k_cache.shape
    most = min(block_table.shape[1] * block_size, cos.shape[0], sin.shape[0])
    for name, t in (("past_seqlens", past_seqlens), ("cache_seqlens", cache_seqlens)):
        if t.device.type != "cpu" and t.device != device:
            raise ValueError(f"{name} must be on the device of q_new (or on the CPU)")
    if cache_seqlens.device.type == "cpu":
        for b, n in enumerate(cache_seqlens.tolist()):
            if n < 0 or n > most:
                raise ValueError(f"cache_seqlens[{b}] = {n} is outside [0, {most}]")
        if past_seqlens.device.type == "cpu":
            for b, (p, n) in enumerate(zip(past_seqlens.tolist(), cache_seqlens.tolist())):
                if p < max(0, n - T) or p > n:
                    raise ValueError(f"past_seqlens[{b}] = {p} is outside [{max(0, n - T)}, {n}]")
        if block_table.device.type == "cpu":
            _check_host_table(block_table, cache_seqlens, block_size, num_blocks)
    elif past_seqlens.device.type == "cpu":
        _check_host_lengths("past_seqlens", past_seqlens, most)
    with _OnDevice(device):
        if block_table.device.type == "cpu" and block_table.dtype == torch.int32:
            block_table = block_table.to(device)
        _validate_int32("block_table", block_table, device)
        return block_table, _device_int32(past_seqlens, device), _device_int32(cache_seqlens, device)
