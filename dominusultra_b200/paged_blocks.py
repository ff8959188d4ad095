"""Blocks of the paged 8-bit cache that several requests share: forks, copies and compaction.

The tables of ``dominusultra_b200.paged`` give each request blocks of its own. These calls let requests
share them: beams of a search, several answers to one prompt, a text that begins like another.

* ``dominus_ultra_paged_fork``: requests continue from others (or end, or shrink), whole blocks shared;
* ``dominus_ultra_paged_copy``: the copies of blocks that a fork or a compaction asks for, for one layer's
  cache (the tables serve all layers, so this is called once for each);
* ``dominus_ultra_paged_compact``: the blocks in use moved to the lowest ids.

A step of a beam search is a fork, a copy in every layer, then the step as before
(``dominus_ultra_paged_tables``, ``dominus_ultra_paged_write``, attention). Everything stays on the GPU; no
call waits for it, and each can be captured into a CUDA graph.
"""

from __future__ import annotations

from typing import Tuple

import torch

from . import _lib
from .attention import _OnDevice, _validate_head_dim
from .paged import (
    _GET_DEVICE,
    _check_host_lengths,
    _device_int32,
    _fit_cache,
    _lengths,
    _stream_of,
    _validate_block_size,
    _validate_int32,
    _validate_paged_cache,
    _workspace,
)

__all__ = [
    "dominus_ultra_paged_fork",
    "dominus_ultra_paged_copy",
    "dominus_ultra_paged_compact",
]

_I32 = torch.int32


def _fit_state(block_table, free_blocks, free_state, block_size) -> bool:
    """One look at what a call with tables and a ring has to have."""
    shape, index = block_table.shape, block_table.get_device()
    return (
        len(shape) == 2 and shape[0] > 0 and shape[1] > 0 and index >= 0 and block_size in (16, 32, 64, 128)
        and block_table.dtype is _I32 and block_table.is_contiguous()
        and free_blocks.dtype is _I32 and free_blocks.get_device() == index and free_blocks.is_contiguous()
        and free_state.dtype is _I32 and free_state.get_device() == index and free_state.is_contiguous()
        and free_blocks.dim() == 1 and free_blocks.shape[0] > 0 and free_state.dim() == 1 and free_state.shape[0] == 2
    )


def _fit_ints(t, batch, index) -> bool:
    return t.dtype is _I32 and t.get_device() == index and t.is_contiguous() and t.dim() == 1 and t.shape[0] == batch


def _check_state(block_table, free_blocks, free_state, block_size, lengths) -> torch.device:
    """The refusals of tables, ring and lengths ({name: tensor}); returns the device."""
    if block_table.ndim != 2 or block_table.shape[0] <= 0 or block_table.shape[1] <= 0:
        raise ValueError("block_table must be a non-empty [batch, max_blocks] tensor")
    _validate_block_size(block_size)
    for name, t in lengths.items():
        _lengths(name, t, block_table.shape[0])
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
    for name, t in lengths.items():
        if t.device.type != "cpu" and t.device != device:
            raise ValueError(f"{name} must be on the device of block_table (or on the CPU)")
    return device


def dominus_ultra_paged_fork(
    block_table: torch.Tensor,
    cache_seqlens: torch.Tensor,
    sources: torch.Tensor,
    new_seqlens: torch.Tensor,
    free_blocks: torch.Tensor,
    free_state: torch.Tensor,
    block_size: int,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """
    Requests that continue from others, with shared blocks (``du_paged_fork``).

    Request ``b`` becomes the first ``new_seqlens[b]`` tokens of request ``sources[b]``, all at once
    from the state before the call: beams that change places, several requests from one prompt, a
    request that shrinks (``sources[b] == b``) or ends (length 0). Whole blocks are shared. A last
    block that is partly filled will be written, so it has to be the request's own: the lowest of the
    requests that end in it keeps it, unless some request holds it whole; each of the others takes a free
    block, in order of ``b``, and leaves a pair for ``dominus_ultra_paged_copy``, which must run on
    every layer's cache before the blocks are written or read. A request for which no block is left is
    cut to its whole blocks, as its returned length says. Blocks that nobody holds any more go behind
    the ring's tail in order of their ids, free from the next call on.

    Requests that share blocks shrink and end through this call: ``dominus_ultra_paged_tables`` would
    give back a block that others hold. They grow through ``dominus_ultra_paged_tables`` as ever.

    ``free_blocks`` (given-back ids) is updated in place; everything else is returned: pass it to the
    next call, or copy it into the same tensors inside a captured graph.

    Args:
        block_table: [batch, max_blocks] int32
        cache_seqlens: [batch] integer tokens cached (int32 or int64; on the CPU they are checked
            here, on the GPU a request out of range keeps its row and every block in it, and
            ``_lib.read_status()`` reports 6)
        sources: [batch] integer requests to continue from
        new_seqlens: [batch] integer tokens to take over, at most the source's
        free_blocks: [num_blocks] int32, a ring of free block ids
        free_state: [2] int32, {head, count} of the ring
        block_size: 16, 32, 64 or 128

    Returns:
        Tuple of:
            - block_table: [batch, max_blocks] int32, -1 behind each request's blocks
            - copies: [batch, 2] int32, {source, destination} blocks, -1 where there is none
            - seqlens: [batch] int32, the lengths that the requests have now
            - free_state: [2] int32
    """
    index = block_table.get_device()
    if not (
        _fit_state(block_table, free_blocks, free_state, block_size)
        and _fit_ints(cache_seqlens, block_table.shape[0], index)
        and _fit_ints(sources, block_table.shape[0], index)
        and _fit_ints(new_seqlens, block_table.shape[0], index)
    ):
        cache_seqlens, sources, new_seqlens = _check_fork(
            block_table, cache_seqlens, sources, new_seqlens, free_blocks, free_state, block_size
        )
    if _GET_DEVICE() != index:
        with _OnDevice(block_table.device):
            return dominus_ultra_paged_fork(
                block_table, cache_seqlens, sources, new_seqlens, free_blocks, free_state, block_size
            )
    batch, max_blocks = block_table.shape
    table = torch.empty_like(block_table)
    copies = block_table.new_empty((batch, 2))
    seqlens = torch.empty_like(cache_seqlens)
    state = torch.empty_like(free_state)
    rc = _lib.load().du_paged_fork(
        block_table.data_ptr(), cache_seqlens.data_ptr(), sources.data_ptr(), new_seqlens.data_ptr(),
        free_blocks.data_ptr(), free_state.data_ptr(), table.data_ptr(), copies.data_ptr(), seqlens.data_ptr(),
        state.data_ptr(), batch, max_blocks, free_blocks.shape[0], block_size, _stream_of(index),
    )
    if rc:
        _lib.check(rc, "du_paged_fork")
    return table, copies, seqlens, state


def _check_fork(block_table, cache_seqlens, sources, new_seqlens, free_blocks, free_state, block_size):
    """The refusals of dominus_ultra_paged_fork; returns lengths and sources as int32 on the device."""
    named = {"cache_seqlens": cache_seqlens, "sources": sources, "new_seqlens": new_seqlens}
    device = _check_state(block_table, free_blocks, free_state, block_size, named)
    batch, max_blocks = block_table.shape
    for name, hi in (("cache_seqlens", max_blocks * block_size), ("sources", batch - 1), ("new_seqlens", max_blocks * block_size)):
        if named[name].device.type == "cpu":
            _check_host_lengths(name, named[name], hi)
    with _OnDevice(device):
        return tuple(_device_int32(t, device) for t in named.values())


def dominus_ultra_paged_copy(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    copies: torch.Tensor,
) -> None:
    """
    Copy blocks of the paged 8-bit cache, keys, values and scales, in place (``du_paged_copy``).

    A block must not be the destination of two pairs, nor the source of one and the destination of
    another (those of a fork or of a compaction never are). A pair with a block id out of range is left
    out, and ``_lib.read_status()`` reports code 7.

    Args:
        k_cache, v_cache: [num_blocks, num_kv_heads, block_size, head_dim] float8_e4m3fn
        k_scale, v_scale: [num_blocks, num_kv_heads] fp32
        copies: [n, 2] int32 {source, destination} blocks, -1 where there is none
    """
    cache, index = k_cache.shape, k_cache.get_device()
    if not (
        len(cache) == 4 and index >= 0 and cache[3] in (16, 32, 64, 128, 256)
        and _fit_cache(k_cache, v_cache, k_scale, v_scale, cache, index)
        and copies.dtype is _I32 and copies.get_device() == index and copies.is_contiguous()
        and copies.dim() == 2 and copies.shape[1] == 2
    ):
        _check_copy(k_cache, v_cache, k_scale, v_scale, copies)
    if _GET_DEVICE() != index:
        with _OnDevice(k_cache.device):
            return dominus_ultra_paged_copy(k_cache, v_cache, k_scale, v_scale, copies)
    rc = _lib.load().du_paged_copy(
        k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), copies.data_ptr(),
        copies.shape[0], *cache, _stream_of(index),
    )
    if rc:
        _lib.check(rc, "du_paged_copy")


def _check_copy(k_cache, v_cache, k_scale, v_scale, copies) -> None:
    """The refusals of dominus_ultra_paged_copy."""
    if k_cache.ndim != 4 or v_cache.ndim != 4:
        raise ValueError("k_cache and v_cache must be rank-4 tensors")
    if copies.ndim != 2 or copies.shape[1] != 2:
        raise ValueError("copies must have shape [n, 2]")
    _validate_head_dim(k_cache.shape[3])
    if not k_cache.is_cuda:
        raise ValueError("DominusUltra kernels require CUDA tensors")
    _validate_paged_cache(k_cache, v_cache, k_scale, v_scale, k_cache.device)
    _validate_int32("copies", copies, k_cache.device)


def dominus_ultra_paged_compact(
    block_table: torch.Tensor,
    cache_seqlens: torch.Tensor,
    free_blocks: torch.Tensor,
    free_state: torch.Tensor,
    block_size: int,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """
    Move the blocks in use to the lowest ids (``du_paged_compact``).

    Of the blocks that these requests hold and the free ones, the lowest ids become the ones in use, so
    that what lies behind them can be given up: blocks above move into the free ones below, both in
    ascending order. Blocks in neither set belong to others and stay. The pairs are for
    ``dominus_ultra_paged_copy``, which must run on every layer's cache before it is read or written.
    Nothing is updated in place.

    Args:
        block_table: [batch, max_blocks] int32
        cache_seqlens: [batch] integer tokens cached (int32 or int64; on the CPU they are checked
            here, on the GPU a request out of range keeps its row, every block in it stays where it is,
            and ``_lib.read_status()`` reports 6)
        free_blocks: [num_blocks] int32, a ring of free block ids
        free_state: [2] int32, {head, count} of the ring; if that does not hold ``count`` different
            blocks that nobody uses, nothing moves, and the status is 7
        block_size: 16, 32, 64 or 128

    Returns:
        Tuple of:
            - block_table: [batch, max_blocks] int32, -1 behind each request's blocks
            - copies: [num_blocks // 2, 2] int32, {source, destination} blocks, then -1
            - free_blocks: [num_blocks] int32, the free ids in ascending order, then -1
            - free_state: [2] int32
    """
    index = block_table.get_device()
    if not (
        _fit_state(block_table, free_blocks, free_state, block_size)
        and _fit_ints(cache_seqlens, block_table.shape[0], index)
    ):
        cache_seqlens = _check_compact(block_table, cache_seqlens, free_blocks, free_state, block_size)
    if _GET_DEVICE() != index:
        with _OnDevice(block_table.device):
            return dominus_ultra_paged_compact(block_table, cache_seqlens, free_blocks, free_state, block_size)
    batch, max_blocks = block_table.shape
    num_blocks = free_blocks.shape[0]
    table = torch.empty_like(block_table)
    copies = block_table.new_empty((num_blocks // 2, 2))
    ring = torch.empty_like(free_blocks)
    state = torch.empty_like(free_state)
    stream = _stream_of(index)
    nbytes = 16 * (1 + (num_blocks + 127) // 128 * 4)  # (du_paged_compact_workspace_size, which a test compares)
    ws, keep = _workspace(nbytes, index, stream)
    rc = _lib.load().du_paged_compact(
        block_table.data_ptr(), cache_seqlens.data_ptr(), free_blocks.data_ptr(), free_state.data_ptr(),
        table.data_ptr(), copies.data_ptr(), ring.data_ptr(), state.data_ptr(), batch, max_blocks, num_blocks,
        block_size, ws, nbytes, stream,
    )
    if rc:
        _lib.check(rc, "du_paged_compact")
    return table, copies, ring, state


def _check_compact(block_table, cache_seqlens, free_blocks, free_state, block_size):
    """The refusals of dominus_ultra_paged_compact; returns the lengths as int32 on the device."""
    device = _check_state(block_table, free_blocks, free_state, block_size, {"cache_seqlens": cache_seqlens})
    if cache_seqlens.device.type == "cpu":
        _check_host_lengths("cache_seqlens", cache_seqlens, block_table.shape[1] * block_size)
    with _OnDevice(device):
        return _device_int32(cache_seqlens, device)
