"""Batches whose requests fill the attention's CTAs with many chunks each: sizes only (the CPU tests look
at how the kernel splits them, the GPU tests run them)."""

from __future__ import annotations

import random

import torch

BF16, F16 = torch.bfloat16, torch.float16


def _lens(seed, count, low, high):
    r = random.Random(seed)
    return [r.randint(low, high) for _ in range(count)]


# name: query heads, KV heads, head_dim, block, lengths, dtype
EQUAL_RANGES = {
    "64 requests, 32 heads on 8 of 128": (32, 8, 128, 16, _lens(1, 64, 600, 3000), BF16),
    "40 requests, 64 heads on 8 of 128": (64, 8, 128, 32, _lens(2, 40, 600, 3000), F16),
    "50 requests, 8 heads of 64": (8, 8, 64, 64, _lens(3, 50, 600, 3000), BF16),
    "45 requests, 16 heads on 8 of 64": (16, 8, 64, 16, _lens(4, 45, 600, 3000), F16),
    "330 requests, 8 heads on one of 32": (8, 1, 32, 16, _lens(5, 330, 600, 1700), BF16),
    "20 requests, 64 heads on 16 of 32": (64, 16, 32, 64, _lens(6, 20, 600, 2900), BF16),
    "160 requests, 4 heads on 2 of 256": (4, 2, 256, 16, _lens(7, 160, 600, 2500), F16),
    "100 requests, 16 heads on one of 256": (16, 1, 256, 128, _lens(8, 100, 600, 2500), BF16),
    "80 requests, 12 heads on 3 of 256": (12, 3, 256, 32, _lens(9, 80, 600, 2000), BF16),
    "200 requests, 6 heads on 2 of 16": (6, 2, 16, 16, _lens(10, 200, 600, 2500), BF16),
    "400 requests, one head of 128": (1, 1, 128, 128, _lens(11, 400, 600, 2000), F16),
    "16 uneven requests, 64 heads on 8 of 128": (64, 8, 128, 128, [20001, 777] + _lens(12, 14, 100, 20001), F16),
    "36 uneven requests, 32 heads on 8 of 64": (32, 8, 64, 16, [30000, 1, 0, 129] + _lens(13, 32, 1, 5000), BF16),
}
PIECES = {
    "one of 30000, 32 heads on 8 of 128": (32, 8, 128, 16, [30000], BF16),
    "296 requests, one head of 64": (1, 1, 64, 16, _lens(20, 296, 2000, 2048), F16),
    "one of 70000, 2 heads on one of 16": (2, 1, 16, 16, [70000], BF16),
    "one of 50001, 4 heads on one of 256": (4, 1, 256, 64, [50001], BF16),
    "3 of 9000, 24 heads on 3 of 64": (24, 3, 64, 32, [9000, 8999, 8800], F16),
    "2 of 20000, 5 heads on 5 of 32": (5, 5, 32, 128, [20000, 19000], F16),
}
