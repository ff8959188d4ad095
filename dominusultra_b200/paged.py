"""Paged KV cache held in 8 bits: block tables, the cache's writer and its single-token attention.

The serving step around ``dominus_ultra_decode`` (reference ``dominus_ultra.py:504-583``, which
reads one contiguous 16-bit cache of one length) with the cache cut into blocks of tokens and held
as e4m3 with one scale per (block, KV head):

* ``k_cache``, ``v_cache``: ``[num_blocks, num_kv_heads, block_size, head_dim]``
  ``torch.float8_e4m3fn``, ``block_size`` 16, 32, 64 or 128; keys are stored rotated;
* ``k_scale``, ``v_scale``: ``[num_blocks, num_kv_heads]`` fp32;
* ``block_table``: ``[batch, max_blocks]`` int32, the blocks of each request in order.

A step is ``dominus_ultra_paged_tables`` (blocks and slots for the new tokens),
``dominus_ultra_paged_write`` (their keys and values) and ``dominus_ultra_decode_paged``. Lengths
and tables stay on the GPU: a step waits for nothing there, and each call can be captured into a CUDA
graph. Two things do wait: lengths or a table given on the CPU are copied, and the first eager decode on
a device (then the next one after every 512 captured ones) copies 4 MB of zeroed tickets from the host.
"""

from __future__ import annotations

import threading
from typing import Tuple

import torch

from . import _lib
from .attention import (
    _RAW_STREAM,
    _RETIRED,
    _aligned,
    _OnDevice,
    _stream,
    _validate_attention_tensors,
    _validate_head_dim,
)

__all__ = [
    "dominus_ultra_paged_tables",
    "dominus_ultra_paged_write",
    "dominus_ultra_decode_paged",
]


_I32, _I64, _F32, _E4M3 = torch.int32, torch.int64, torch.float32, torch.float8_e4m3fn
_F16, _BF16 = torch.float16, torch.bfloat16
_BLOCK_SIZES = (16, 32, 64, 128)
_HEAD_DIMS = (16, 32, 64, 128, 256)
_CODES = {_F16: _lib.DU_DTYPE_F16, _BF16: _lib.DU_DTYPE_BF16}
_GET_DEVICE = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device




def _stream_of(index: int) -> int:
    """Handle of torch's current stream on the device of this index."""
    return _RAW_STREAM(index) if _RAW_STREAM is not None else _stream(torch.device("cuda", index))


def _validate_block_size(block_size: int) -> None:
    if block_size not in _BLOCK_SIZES:
        raise ValueError("block_size must be 16, 32, 64 or 128")


def _validate_int32(name: str, t: torch.Tensor, device: torch.device) -> None:
    if t.dtype != torch.int32:
        raise ValueError(f"{name} must be an int32 tensor")
    if t.device != device:
        raise ValueError(f"{name} must be on the same CUDA device as the other tensors")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _lengths(name: str, t: torch.Tensor, batch: int) -> None:
    if t.ndim != 1 or t.shape[0] != batch:
        raise ValueError(f"{name} must have shape [batch]")
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be an int32 or int64 tensor")


def _check_host_lengths(name: str, t: torch.Tensor, hi: int) -> None:
    """Range check of lengths that are on the CPU (those on the GPU are checked there)."""
    bad = [(i, n) for i, n in enumerate(t.tolist()) if n < 0 or n > hi]
    if bad:
        raise ValueError(f"{name}[{bad[0][0]}] = {bad[0][1]} is outside [0, {hi}]")


def _check_host_table(table: torch.Tensor, lengths: torch.Tensor, block_size: int, num_blocks: int) -> None:
    """Range check of the block ids that `lengths` tokens use, for a table on the CPU."""
    for b, n in enumerate(lengths.tolist()):
        used = table[b, : -(-n // block_size)]
        bad = ((used < 0) | (used >= num_blocks)).nonzero()
        if bad.numel():
            page = int(bad[0])
            raise ValueError(f"block_table[{b}, {page}] = {int(used[page])} is outside [0, {num_blocks - 1}]")


def _device_int32(t: torch.Tensor, device: torch.device) -> torch.Tensor:
    """Lengths as a contiguous int32 tensor on `device`; 64-bit ones out of int32's range stay out
    of every length's range."""
    if t.dtype == torch.int64:
        t = t.clamp(-1, 2**31 - 1).to(torch.int32)
    return t.to(device).contiguous()


def _validate_paged_cache(k_cache, v_cache, k_scale, v_scale, device) -> None:
    if k_cache.ndim != 4 or v_cache.ndim != 4:
        raise ValueError("k_cache and v_cache must be rank-4 tensors")
    num_blocks, hkv, block_size, _ = k_cache.shape
    if v_cache.shape != k_cache.shape:
        raise ValueError("k_cache and v_cache must have the same shape")
    if num_blocks <= 0 or hkv <= 0:
        raise ValueError("num_blocks and num_kv_heads must be positive")
    _validate_block_size(block_size)
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.dtype != torch.float8_e4m3fn:
            raise ValueError(f"{name} must use float8_e4m3fn")
        if t.device != device:
            raise ValueError("all attention tensors must be on the same CUDA device")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if t.data_ptr() % 16:
            raise ValueError(f"{name} must be 16-byte aligned")
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if t.shape != (num_blocks, hkv):
            raise ValueError(f"{name} must have shape [num_blocks, num_kv_heads]")
        if t.dtype != torch.float32:
            raise ValueError(f"{name} must use float32")
        if t.device != device:
            raise ValueError("all attention tensors must be on the same CUDA device")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")


def _validate_tables_like(cos, sin, head_dim, device, dtype) -> None:
    """The rope tables but for their length: the positions are known on the GPU only."""
    expected_tail = (head_dim // 2,)
    if cos.ndim != 2 or sin.ndim != 2:
        raise ValueError("cos and sin must be rank-2 [positions, head_dim // 2] tensors")
    if cos.shape[0] < 1 or sin.shape[0] < 1:
        raise ValueError("cos and sin must contain at least 1 positions")
    if cos.shape[1:] != expected_tail or sin.shape[1:] != expected_tail:
        raise ValueError(f"cos and sin must have trailing shape {expected_tail}")
    if cos.device != device or sin.device != device:
        raise ValueError("cos and sin must be on the same device as the attention tensors")
    if cos.dtype != dtype or sin.dtype != dtype:
        raise ValueError("cos and sin must have the same dtype as the attention tensors")
    if not cos.is_contiguous() or not sin.is_contiguous():
        raise ValueError("cos and sin must be contiguous")


_WS_SIZES = {}


def _decode_workspace_size(B, Hq, Hkv, D, block_size, max_blocks, index) -> int:
    key = (B, Hq, Hkv, D, block_size, max_blocks, index)
    n = _WS_SIZES.get(key)
    if n is None:
        n = int(_lib.load().du_decode_paged_workspace_size(B, Hq, Hkv, D, block_size, max_blocks))
        _WS_SIZES[key] = n
    return n


# Tickets for calls under a graph capture, handed out of zeroed slabs: [slab, words used] per device.
# A captured call's tickets are its own for good; those of graphs that are gone are not taken back, 4 KB
# each. Its workspace is memory of the capture's pool. So any two graphs may be replayed at once, unless
# they were captured into one pool, which torch allows only for graphs that never run together.
_SLAB_WORDS = 1024 * _lib.DU_PAGED_TICKETS
_SLABS = {}
_SLAB_LOCK = threading.Lock()


# Scratch of eager calls per (device, stream): [tickets, workspace], the workspace grown on demand.
_SCRATCH = {}


def _decode_scratch(nbytes: int, index: int, stream: int):
    """(tickets, workspace, what keeps them alive until the launch) of a paged decode on torch's
    current stream.

    Eager calls share a pair per (device, stream): calls on one stream run in order. Another thread's
    call on the stream may replace the pair before this one's launch, and a buffer that nothing
    holds could then be another tensor's. A call that is being captured gets a workspace from the
    graph's own memory and tickets of its own.
    """
    if not torch.cuda.is_current_stream_capturing():
        pair = _SCRATCH.get((index, stream))
        slab = _SLABS.get(index)
        if pair is None or pair[2] < nbytes or slab is None or slab[1] > _SLAB_WORDS // 2:
            pair = _grow_scratch(nbytes, index, stream)
        return pair[0], pair[1], pair
    device = torch.device("cuda", index)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    with _SLAB_LOCK:
        slab = _SLABS.get(index)
        if slab is not None and slab[1] + _lib.DU_PAGED_TICKETS <= _SLAB_WORDS:
            tickets = slab[0].data_ptr() + 4 * slab[1]
            slab[1] += _lib.DU_PAGED_TICKETS
            return tickets, ws.data_ptr(), ws
    # no slab yet (the process's first call), or more than half a slab of captures since the last
    # eager call: zeroed inside the graph, by a node of its own
    tickets = torch.zeros(_lib.DU_PAGED_TICKETS, dtype=torch.int32, device=device)
    return tickets.data_ptr(), ws.data_ptr(), (ws, tickets)


def _grow_scratch(nbytes: int, index: int, stream: int):
    """A (device, stream)'s scratch of at least nbytes, and a ticket slab with room for captures."""
    device = torch.device("cuda", index)
    with _SLAB_LOCK:
        slab = _SLABS.get(index)
        if slab is None or slab[1] > _SLAB_WORDS // 2:
            if slab is not None:
                _RETIRED.append(slab[0])  # graphs count in it
            # (a copy from the host has ended when it returns: the zeros are there for any stream)
            _SLABS[index] = [torch.zeros(_SLAB_WORDS, dtype=torch.int32).to(device), 0]
        pair = _SCRATCH.get((index, stream))
        if pair is None or pair[2] < nbytes:
            size = max(nbytes, 2 * pair[2] if pair is not None else 0)
            tickets = pair[3] if pair is not None else torch.zeros(_lib.DU_PAGED_TICKETS, dtype=torch.int32, device=device)
            ws = torch.empty(size, dtype=torch.uint8, device=device)
            pair = (tickets.data_ptr(), ws.data_ptr(), size, tickets, ws)
            _SCRATCH[(index, stream)] = pair
    return pair


def dominus_ultra_paged_tables(
    block_table: torch.Tensor,
    cache_seqlens: torch.Tensor,
    new_seqlens: torch.Tensor,
    free_blocks: torch.Tensor,
    free_state: torch.Tensor,
    block_size: int,
    max_new: int,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """
    Block tables and slot map of a step, from the requests' lengths (``du_paged_tables``).

    Request ``b`` holds ``cache_seqlens[b]`` tokens and wants ``new_seqlens[b]``: more (up to
    ``max_new`` more), fewer (a rejected draft), or 0 (a request that ends). Requests that grow
    over a block's end take blocks from the ring of free ones, in order of ``b`` from its head, as
    long as the needs up to a request are covered; a request that is not served keeps its length.
    Requests that shrink give blocks back behind the ring's tail, free from the next call on; a block is
    held by one request only (a block in two rows would be given back twice).

    ``block_table`` (new entries) and ``free_blocks`` (given-back ids) are updated in place; the
    lengths and ``free_state`` are not: pass the returned ones to the next call, or copy them
    into the same tensors inside a captured graph.

    Args:
        block_table: [batch, max_blocks] int32
        cache_seqlens: [batch] integer tokens cached (int32 or int64; on the CPU they are checked
            here, on the GPU a bad request is left as it is and ``_lib.read_status()`` reports 6;
            a table entry that is not a block id is reported as 7 when it is used or given back)
        new_seqlens: [batch] integer tokens wanted
        free_blocks: [num_blocks] int32, a ring of free block ids
        free_state: [2] int32, {head, count} of the ring
        block_size: 16, 32, 64 or 128
        max_new: columns of the slot map

    Returns:
        Tuple of:
            - slots: [batch, max_new] int32, ``block * block_size + row`` of each new token, -1
              where there is none
            - seqlens: [batch] int32, the lengths that the requests have now
            - free_state: [2] int32
    """
    shape = block_table.shape
    index = block_table.get_device()
    # One look at what every call has to have (written out: a call's host time is mostly this); where
    # it fails, the checks by name.
    if not (
        len(shape) == 2 and shape[0] > 0 and shape[1] > 0 and index >= 0
        and block_size in _BLOCK_SIZES and max_new >= 0
        and block_table.dtype is _I32 and block_table.is_contiguous()
        and free_blocks.dtype is _I32 and free_blocks.get_device() == index and free_blocks.is_contiguous()
        and free_state.dtype is _I32 and free_state.get_device() == index and free_state.is_contiguous()
        and free_blocks.dim() == 1 and free_blocks.shape[0] > 0 and free_state.dim() == 1 and free_state.shape[0] == 2
        and cache_seqlens.dtype is _I32 and cache_seqlens.get_device() == index and cache_seqlens.is_contiguous()
        and new_seqlens.dtype is _I32 and new_seqlens.get_device() == index and new_seqlens.is_contiguous()
        and cache_seqlens.dim() == 1 and cache_seqlens.shape[0] == shape[0]
        and new_seqlens.dim() == 1 and new_seqlens.shape[0] == shape[0]
    ):
        cache_seqlens, new_seqlens = _check_tables(
            block_table, cache_seqlens, new_seqlens, free_blocks, free_state, block_size, max_new
        )
    if _GET_DEVICE() != index:
        with _OnDevice(block_table.device):
            return dominus_ultra_paged_tables(
                block_table, cache_seqlens, new_seqlens, free_blocks, free_state, block_size, max_new
            )
    batch, max_blocks = shape
    slots = block_table.new_empty((batch, max_new))
    seqlens = torch.empty_like(cache_seqlens)
    state = torch.empty_like(free_state)
    rc = _lib.load().du_paged_tables(
        block_table.data_ptr(), cache_seqlens.data_ptr(), new_seqlens.data_ptr(), free_blocks.data_ptr(),
        free_state.data_ptr(), slots.data_ptr(), seqlens.data_ptr(), state.data_ptr(), batch, max_blocks,
        free_blocks.shape[0], block_size, max_new, _stream_of(index),
    )
    if rc:
        _lib.check(rc, "du_paged_tables")
    return slots, seqlens, state


def _check_tables(block_table, cache_seqlens, new_seqlens, free_blocks, free_state, block_size, max_new):
    """The refusals of dominus_ultra_paged_tables; returns the lengths as int32 on the device."""
    if block_table.ndim != 2 or block_table.shape[0] <= 0 or block_table.shape[1] <= 0:
        raise ValueError("block_table must be a non-empty [batch, max_blocks] tensor")
    batch, max_blocks = block_table.shape
    _validate_block_size(block_size)
    if max_new < 0:
        raise ValueError("max_new must not be negative")
    _lengths("cache_seqlens", cache_seqlens, batch)
    _lengths("new_seqlens", new_seqlens, batch)
    if free_blocks.ndim != 1 or free_blocks.shape[0] <= 0:
        raise ValueError("free_blocks must be a non-empty [num_blocks] tensor")
    if free_state.shape != (2,):
        raise ValueError("free_state must have shape [2]")
    if not block_table.is_cuda:
        raise ValueError("DominusUltra kernels require CUDA tensors")
    device = block_table.device
    _validate_int32("block_table", block_table, device)
    _validate_int32("free_blocks", free_blocks, device)
    _validate_int32("free_state", free_state, device)
    for name, t in (("cache_seqlens", cache_seqlens), ("new_seqlens", new_seqlens)):
        if t.device.type == "cpu":
            _check_host_lengths(name, t, max_blocks * block_size)
        elif t.device != device:
            raise ValueError(f"{name} must be on the device of block_table (or on the CPU)")
    with _OnDevice(device):
        return _device_int32(cache_seqlens, device), _device_int32(new_seqlens, device)


def dominus_ultra_paged_write(
    k_new: torch.Tensor,
    v_new: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    slots: torch.Tensor,
    cache_seqlens: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
) -> None:
    """
    Write new tokens' keys and values into the paged 8-bit cache, in place (``du_paged_write``).

    Token ``t`` of request ``b`` rotates at position ``cache_seqlens[b] + t`` and goes to
    ``slots[b, t]``. Each (block, KV head) of keys and of values has a scale, a power of two: the
    smallest that covers the rows written, or the present one where the block holds earlier rows
    and theirs is larger; when it grows, the earlier rows are rescaled. Values are rounded once, to
    the nearest e4m3 value. A value that is not finite makes its block's scale NaN.

    Requests must not share a block that they write to. (Blocks that are only read may be shared by the
    attention; ``dominus_ultra_paged_tables`` counts no references to them.)

    Args:
        k_new, v_new: [batch, num_kv_heads, T, head_dim], keys not rotated (one token each, or
            whole prompts as ``dominus_ultra_prefill`` takes them)
        k_cache, v_cache: [num_blocks, num_kv_heads, block_size, head_dim] float8_e4m3fn
        k_scale, v_scale: [num_blocks, num_kv_heads] fp32
        slots: [batch, T] int32 from ``dominus_ultra_paged_tables``, -1 for no token
        cache_seqlens: [batch] integer lengths before these tokens (what the tables call took)
        cos, sin: tables from precompute_rope_cos_sin covering the new positions
    """
    shape, cache = k_new.shape, k_cache.shape
    index, dtype = k_new.get_device(), k_new.dtype
    if not (
        len(shape) == 4 and len(cache) == 4 and index >= 0 and dtype in _CODES
        and k_new.is_contiguous() and v_new.shape == shape
        and v_new.dtype is dtype and v_new.get_device() == index and v_new.is_contiguous()
        and _fit_rope(cos, sin, dtype, index, shape[3])
        and shape[0] > 0 and shape[1] > 0 and shape[2] > 0 and shape[3] in _HEAD_DIMS
        and _fit_cache(k_cache, v_cache, k_scale, v_scale, cache, index)
        and cache[1] == shape[1] and cache[3] == shape[3]
        and slots.dtype is _I32 and slots.get_device() == index and slots.is_contiguous()
        and slots.dim() == 2 and slots.shape[0] == shape[0] and slots.shape[1] == shape[2]
        and cache_seqlens.dtype is _I32 and cache_seqlens.get_device() == index and cache_seqlens.is_contiguous()
        and cache_seqlens.dim() == 1 and cache_seqlens.shape[0] == shape[0]
    ):
        cache_seqlens = _check_write(k_new, v_new, k_cache, v_cache, k_scale, v_scale, slots, cache_seqlens, cos, sin)
    if _GET_DEVICE() != index:
        with _OnDevice(k_new.device):
            return dominus_ultra_paged_write(
                k_new, v_new, k_cache, v_cache, k_scale, v_scale, slots, cache_seqlens, cos, sin
            )
    k, v, c, s = k_new.data_ptr(), v_new.data_ptr(), cos.data_ptr(), sin.data_ptr()
    if (k | v | c | s) & 15:
        k_new, v_new, cos, sin = (_aligned(t) for t in (k_new, v_new, cos, sin))
        k, v, c, s = k_new.data_ptr(), v_new.data_ptr(), cos.data_ptr(), sin.data_ptr()
    rc = _lib.load().du_paged_write(
        k, v, k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), slots.data_ptr(),
        cache_seqlens.data_ptr(), c, s, *shape, cache[0], cache[2], _CODES[dtype],
        min(cos.shape[0], sin.shape[0]), _stream_of(index),
    )
    if rc:
        _lib.check(rc, "du_paged_write")


def _fit_rope(cos, sin, dtype, index, head_dim) -> bool:
    c, s = cos.shape, sin.shape
    return (
        cos.dtype is dtype and cos.get_device() == index and cos.is_contiguous()
        and sin.dtype is dtype and sin.get_device() == index and sin.is_contiguous()
        and len(c) == 2 and len(s) == 2 and c[1] * 2 == head_dim and s[1] * 2 == head_dim and c[0] > 0 and s[0] > 0
    )


def _fit_cache(k_cache, v_cache, k_scale, v_scale, cache, index) -> bool:
    pair = cache[:2]
    return (
        k_cache.dtype is _E4M3 and k_cache.get_device() == index and k_cache.is_contiguous()
        and v_cache.dtype is _E4M3 and v_cache.get_device() == index and v_cache.is_contiguous()
        and v_cache.shape == cache and cache[0] > 0 and cache[1] > 0 and cache[2] in _BLOCK_SIZES
        and not (k_cache.data_ptr() | v_cache.data_ptr()) & 15
        and k_scale.dtype is _F32 and k_scale.get_device() == index and k_scale.is_contiguous()
        and v_scale.dtype is _F32 and v_scale.get_device() == index and v_scale.is_contiguous()
        and k_scale.shape == pair and v_scale.shape == pair
    )


def _check_write(k_new, v_new, k_cache, v_cache, k_scale, v_scale, slots, cache_seqlens, cos, sin):
    """The refusals of dominus_ultra_paged_write; returns the lengths as int32 on the device."""
    if k_new.ndim != 4 or v_new.ndim != 4 or k_cache.ndim != 4 or v_cache.ndim != 4:
        raise ValueError("k_new, v_new, k_cache, and v_cache must be rank-4 tensors")
    B, Hkv, T, D = k_new.shape
    if B <= 0 or Hkv <= 0 or T <= 0:
        raise ValueError("batch, heads, and sequence length must be positive")
    if v_new.shape != k_new.shape:
        raise ValueError("k_new and v_new must have the same shape")
    if k_cache.shape[1] != Hkv or k_cache.shape[3] != D:
        raise ValueError("the caches must have k_new's head count and head_dim")
    if slots.shape != (B, T):
        raise ValueError("slots must have shape [batch, T]")
    _lengths("cache_seqlens", cache_seqlens, B)
    _validate_head_dim(D)
    _validate_attention_tensors(k_new, v_new)
    device = k_new.device
    _validate_paged_cache(k_cache, v_cache, k_scale, v_scale, device)
    _validate_int32("slots", slots, device)
    _validate_tables_like(cos, sin, D, device, k_new.dtype)
    if cache_seqlens.device.type == "cpu":
        _check_host_lengths("cache_seqlens", cache_seqlens, min(cos.shape[0], sin.shape[0]))
    elif cache_seqlens.device != device:
        raise ValueError("cache_seqlens must be on the device of k_new (or on the CPU)")
    with _OnDevice(device):
        return _device_int32(cache_seqlens, device)


def dominus_ultra_decode_paged(
    q_new: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_table: torch.Tensor,
    cache_seqlens: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
) -> torch.Tensor:
    """
    Decode-phase attention over the paged 8-bit cache (``du_decode_paged``).

    ``cache_seqlens[b]`` counts the cached tokens with the new one (what
    ``dominus_ultra_paged_tables`` returned, after ``dominus_ultra_paged_write``): the query
    rotates at ``cache_seqlens[b] - 1`` and attends to keys ``0..cache_seqlens[b] - 1``, as
    ``dominus_ultra_decode_kvcache`` does with an append. A request of length 0 gives zeros. Rows of
    a block behind the length are never used, whatever they hold.

    Lengths and table are read on the GPU: a length out of range gives zeros, a block id out of
    range NaN, and ``_lib.read_status()`` reports code 6 or 7. Given on the CPU, they are checked
    here.

    Args:
        q_new: [batch, num_heads, 1, head_dim]
        k_cache, v_cache: [num_blocks, num_kv_heads, block_size, head_dim] float8_e4m3fn
        k_scale, v_scale: [num_blocks, num_kv_heads] fp32, positive
        block_table: [batch, max_blocks] int32
        cache_seqlens: [batch] integer lengths
        cos, sin: tables from precompute_rope_cos_sin covering every length

    Returns:
        Output tensor of shape [batch, num_heads, 1, head_dim]
    """
    shape, cache, table = q_new.shape, k_cache.shape, block_table.shape
    index, dtype = q_new.get_device(), q_new.dtype
    if not (
        len(shape) == 4 and len(cache) == 4 and len(table) == 2 and index >= 0 and dtype in _CODES
        and q_new.is_contiguous() and _fit_rope(cos, sin, dtype, index, shape[3])
        and shape[0] > 0 and shape[1] > 0 and shape[2] == 1 and shape[3] in _HEAD_DIMS
        and _fit_cache(k_cache, v_cache, k_scale, v_scale, cache, index)
        and shape[1] % cache[1] == 0 and cache[3] == shape[3]
        and block_table.dtype is _I32 and block_table.get_device() == index and block_table.is_contiguous()
        and table[0] == shape[0] and table[1] > 0
        and cache_seqlens.dtype is _I32 and cache_seqlens.get_device() == index and cache_seqlens.is_contiguous()
        and cache_seqlens.dim() == 1 and cache_seqlens.shape[0] == shape[0]
    ):
        block_table, cache_seqlens = _check_decode(
            q_new, k_cache, v_cache, k_scale, v_scale, block_table, cache_seqlens, cos, sin
        )
    if _GET_DEVICE() != index:
        with _OnDevice(q_new.device):
            return dominus_ultra_decode_paged(
                q_new, k_cache, v_cache, k_scale, v_scale, block_table, cache_seqlens, cos, sin
            )
    B, Hq, _, D = shape
    num_blocks, Hkv, block_size, _ = cache
    max_blocks = table[1]
    q, c, s = q_new.data_ptr(), cos.data_ptr(), sin.data_ptr()
    if (q | c | s) & 15:
        q_new, cos, sin = (_aligned(t) for t in (q_new, cos, sin))
        q, c, s = q_new.data_ptr(), cos.data_ptr(), sin.data_ptr()
    out = torch.empty_like(q_new)
    stream = _stream_of(index)
    nbytes = _decode_workspace_size(B, Hq, Hkv, D, block_size, max_blocks, index)
    tickets, ws, keep = _decode_scratch(nbytes, index, stream)
    rc = _lib.load().du_decode_paged(
        q, k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), block_table.data_ptr(),
        cache_seqlens.data_ptr(), c, s, out.data_ptr(), B, Hq, Hkv, D, num_blocks, block_size, max_blocks,
        _CODES[dtype], D**-0.5, min(cos.shape[0], sin.shape[0]), tickets, ws, nbytes, stream,
    )
    del keep
    if rc:
        _lib.check(rc, "du_decode_paged")
    return out


def _check_decode(q_new, k_cache, v_cache, k_scale, v_scale, block_table, cache_seqlens, cos, sin):
    """The refusals of dominus_ultra_decode_paged; returns the table and the lengths on the device."""
    if q_new.ndim != 4 or k_cache.ndim != 4 or v_cache.ndim != 4:
        raise ValueError("q_new, k_cache, and v_cache must be rank-4 tensors")
    B, Hq, _, D = q_new.shape
    if q_new.shape[2] != 1:
        raise ValueError("q_new must contain exactly one sequence position")
    if B <= 0 or Hq <= 0:
        raise ValueError("batch and heads must be positive")
    Hkv = k_cache.shape[1]
    if Hkv <= 0 or Hq % Hkv != 0:
        raise ValueError("num_query_heads must be divisible by num_kv_heads")
    if k_cache.shape[3] != D:
        raise ValueError("the caches must have q_new's head_dim")
    if block_table.ndim != 2 or block_table.shape[0] != B or block_table.shape[1] <= 0:
        raise ValueError("block_table must have shape [batch, max_blocks]")
    _lengths("cache_seqlens", cache_seqlens, B)
    _validate_head_dim(D)
    _validate_attention_tensors(q_new)
    device = q_new.device
    _validate_paged_cache(k_cache, v_cache, k_scale, v_scale, device)
    _validate_tables_like(cos, sin, D, device, q_new.dtype)
    num_blocks, _, block_size, _ = k_cache.shape
    positions = min(cos.shape[0], sin.shape[0])
    if cache_seqlens.device.type == "cpu":
        _check_host_lengths("cache_seqlens", cache_seqlens, min(block_table.shape[1] * block_size, positions))
        if block_table.device.type == "cpu":
            _check_host_table(block_table, cache_seqlens, block_size, num_blocks)
    elif cache_seqlens.device != device:
        raise ValueError("cache_seqlens must be on the device of q_new (or on the CPU)")
    with _OnDevice(device):
        if block_table.device.type == "cpu" and block_table.dtype == torch.int32:
            block_table = block_table.to(device)
        _validate_int32("block_table", block_table, device)
        return block_table, _device_int32(cache_seqlens, device)
