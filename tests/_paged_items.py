"""How the paged extension cuts a call's rows and keys over its CTAs, where its warps keep query rows and outputs in
shared memory, and batches whose CTAs have several items each."""

from __future__ import annotations

import random

import torch

BF16, F16 = torch.bfloat16, torch.float16


def plan(T, G, D):
    """(row tiles of an item, copies of its rows, keys of a tile, charge of an item's beginning)."""
    tiles = 2 if T * G > 128 and D <= 128 else 1
    copies = 1 if T * G > 64 or D == 256 else 2 if T * G > 32 else 4
    keys = 64 if tiles == 2 or D == 256 else 128
    return tiles, copies, keys, 6 if keys == 64 else 5


def split(past, new, Hq, Hkv, D, T, sms=148):
    """The kernel's fragments: a list per CTA of (request, KV head, item, rows, first tile, end tile, fragments)."""
    G = Hq // Hkv
    row_tiles, _, keys, charge = plan(T, G, D)
    size = 128 * row_tiles
    items = []
    for b, (m, n) in enumerate(zip(past, new)):
        for i in range(-(-n * G // size)):
            rows = min(n * G - i * size, size)
            items += [(b, h, i, rows, (m + (i * size + rows - 1) // G) // keys + 1) for h in range(Hkv)]
    per = max(-(-sum(x[4] + charge for x in items) // sms), charge)
    ctas = [[] for _ in range(sms)]
    at = 0
    for b, h, i, rows, tiles in items:
        first, end = at + charge, at + charge + tiles
        count = (end - 1) // per - first // per + 1
        for c in range(first // per, (end - 1) // per + 1):
            lo, hi = max(first, c * per), min(end, (c + 1) * per)
            ctas[c].append((b, h, i, rows, lo - first, hi - first, count))
        at = end
    return ctas


def offset(row, piece, D):
    """Bytes from the row tile's beginning to 16 bytes of one of its 128 query rows."""
    span = min(128, 2 * D)
    lin = row * span + piece % (span // 16) * 16
    return piece // (span // 16) * 128 * span + (lin ^ ((lin >> 7) & (span // 16 - 1)) << 4)


def _new(seed, count, choices):
    r = random.Random(seed)
    return [r.choice(choices) for _ in range(count)], [r.randint(0, 200) for _ in range(count)]


# name: query heads, KV heads, head_dim, most new tokens, new tokens, tokens before them, dtype
UNCUT = {
    "64 prompts, 32 heads on 8 of 128": (32, 8, 128, 300, *_new(1, 64, [20, 40, 56, 300]), BF16),
    "64 prompts, 32 heads on 8 of 128, fp16": (32, 8, 128, 300, *_new(2, 64, [20, 40, 56, 300]), F16),
    "64 of 40, 32 heads on 8 of 128": (32, 8, 128, 40, [40] * 64, [100] * 64, BF16),
    "64 of 75, 32 heads on 8 of 128": (32, 8, 128, 75, [75] * 64, [225] * 64, F16),
    "64 prompts, 8 heads on 2 of 256": (8, 2, 256, 300, *_new(3, 64, [20, 40, 56, 300]), BF16),
    "96 drafts and prompts, 8 heads on 2 of 256": (8, 2, 256, 56, *_new(4, 96, [1, 5, 20, 40, 56]), F16),
    "300 of 20, 4 heads on 2 of 256": (4, 2, 256, 20, [20] * 300, [64] * 300, BF16),
    "64 prompts, 32 heads on 8 of 64": (32, 8, 64, 300, *_new(5, 64, [20, 40, 56, 300]), BF16),
    "96 prompts, 6 heads on 2 of 32": (6, 2, 32, 150, *_new(6, 96, [11, 33, 50, 150]), F16),
    "96 prompts, 8 heads of 16": (8, 8, 16, 300, *_new(7, 96, [20, 150, 230, 300]), BF16),
    "64 drafts, 32 heads on 8 of 128": (32, 8, 128, 20, *_new(8, 64, [1, 5, 13, 20]), BF16),
}
