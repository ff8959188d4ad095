"""Plain implementations of the paged 8-bit cache operators, in Python integers and 64-bit floats on
the CPU, and the error bound of the attention's outputs."""

from __future__ import annotations

import math

import torch

E4M3_VALUES = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()  # 0 .. 448


def pages(n: int, block: int) -> int:
    return -(-n // block)


def tables(table, old, new, ring, state, block, max_new):
    """One call of the block tables on lists: table [B][width], ring [N], state [head, count].

    Updates table and ring; returns (slots, lengths, state)."""
    head, count = state
    n = len(ring)
    cap = len(table[0]) * block
    ok = 0 <= head < n and 0 <= count <= n
    wish = []
    for o, w in zip(old, new):
        bad = not (0 <= o <= cap and 0 <= w <= cap) or w - o > max_new
        wish.append(o if bad else w)
    held = lambda x: pages(min(max(x, 0), cap), block)  # noqa: E731
    if not ok or count + sum(max(0, held(o) - held(w)) for o, w in zip(old, wish)) > n:
        wish, ok = list(old), False
    taken, sum_need, back, lengths, slots = 0, 0, [], [], []
    for b, (o, w) in enumerate(zip(old, wish)):
        need = max(0, held(w) - held(o))
        sum_need += need
        served = need == 0 or sum_need <= count
        if served:
            for i in range(need):
                table[b][held(o) + i] = ring[(head + taken) % n]
                taken += 1
            back += [table[b][i] for i in range(held(w), held(o))]
        lengths.append(w if served else o)
        row = []
        for t in range(max_new):
            pos = o + t
            row.append(table[b][pos // block] * block + pos % block if served and pos < w else -1)
        slots.append(row)
    for i, x in enumerate(back):
        ring[(head + count + i) % n] = x
    return slots, lengths, [(head + taken) % n, count - taken + len(back)] if ok else [head, count]


def nearest_e4m3(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 magnitude with x's sign, ties to the even last bit (|x| <= 448)."""
    a = x.abs().contiguous()
    hi = torch.searchsorted(E4M3_VALUES, a).clamp(1, 126)
    lo_v, hi_v = E4M3_VALUES[hi - 1], E4M3_VALUES[hi]
    low = (a - lo_v < hi_v - a) | ((a - lo_v == hi_v - a) & ((hi - 1) % 2 == 0))
    return torch.where(low, lo_v, hi_v) * torch.sign(x)


def unit_of(amax: float) -> float:
    """The smallest power of two, 2^-64 at least, whose 448-fold covers amax; NaN if not finite."""
    if not math.isfinite(amax):
        return math.nan
    e = -64
    while 448.0 * 2.0**e < amax:
        e += 1
    return 2.0**e


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Half-split rotation of [..., D] in 64 bits with table rows [..., D/2]."""
    d = x.shape[-1] // 2
    a, b, c, s = x[..., :d].double(), x[..., d:].double(), cos.double(), sin.double()
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def write(k_new, v_new, k8, v8, ks, vs, slots, past, cos, sin):
    """The writer on CPU tensors: k8, v8 64-bit e4m3 values [N, Hkv, block, D] and ks, vs 64-bit
    scales [N, Hkv], updated in place."""
    B, Hkv, T, _ = k_new.shape
    block = k8.shape[2]
    for b in range(B):
        t = 0
        while t < T:
            if slots[b][t] < 0:
                t += 1
                continue
            blk, r = divmod(slots[b][t], block)
            m = 1
            while t + m < T and r + m < block and slots[b][t + m] == slots[b][t] + m:
                m += 1
            for h in range(Hkv):
                p = torch.arange(past[b] + t, past[b] + t + m)
                for x, cache, scale in (
                    (rotate(k_new[b, h, t : t + m], cos[p], sin[p]), k8, ks),
                    (v_new[b, h, t : t + m].double(), v8, vs),
                ):
                    unit = unit_of(x.abs().max().item() if torch.isfinite(x).all() else math.inf)
                    had = scale[blk, h].item()
                    if r > 0 and (math.isnan(had) or not unit > had) and not math.isnan(unit):
                        unit = had
                    if r > 0 and unit > had:
                        cache[blk, h, :r] = nearest_e4m3(cache[blk, h, :r] * (had / unit))
                    cache[blk, h, r : r + m] = nearest_e4m3(x / unit) if not math.isnan(unit) else math.nan
                    scale[blk, h] = unit
            t += m


def attend(q, k8, v8, ks, vs, table, lens, cos, sin):
    """(out [B, Hq, 1, D] in 64 bits, bound): bound is what a kernel's output may be off before its
    last rounding.

    The kernel's scores may be off by d = 2^-12 A + 2^-14 A, A = sum_i |q_i k_i| scale: the query
    elements are carried with at least 12 significant bits (half a step: 2^-12), and 2^-14 A is left
    for the accumulation of the products. Weights are carried as 16-bit values (2^-11) in parts
    that lose at most 2^-12 more, times their own accumulation (2^-12): eps = expm1(d) + 2^-10. A
    weight's parts end at an absolute 2^-18 where the largest is at least 1, so n weights may lose
    n 2^-18 together. With w_j (1 + eps_j) in numerator and denominator the quotient moves by at
    most 2 eps / (1 - eps) sum_j p_j |v_j|, and the lost weights by n 2^-18 max |v|.
    """
    B, Hq, _, D = q.shape
    Hkv, block = k8.shape[1], k8.shape[2]
    G = Hq // Hkv
    out = torch.zeros(B, Hq, 1, D, dtype=torch.float64)
    bound = torch.zeros_like(out)
    scale = D**-0.5
    for b, n in enumerate(lens):
        if n == 0:
            continue
        ids = torch.tensor(table[b][: pages(n, block)])
        qr = rotate(q[b, :, 0], cos[n - 1], sin[n - 1])
        for h in range(Hkv):
            k = (k8[ids, h] * ks[ids, h][:, None, None]).reshape(-1, D)[:n]
            v = (v8[ids, h] * vs[ids, h][:, None, None]).reshape(-1, D)[:n]
            qh = qr[h * G : (h + 1) * G]
            p = torch.softmax(qh @ k.T * scale, -1)
            a = (qh.abs() @ k.abs().T * scale).amax(-1, keepdim=True)
            d = a * (2.0**-12 + 2.0**-14)
            eps = torch.expm1(d) + 2.0**-10
            out[b, h * G : (h + 1) * G, 0] = p @ v
            bound[b, h * G : (h + 1) * G, 0] = 2 * eps / (1 - eps) * (p @ v.abs()) + n * 2.0**-18 * v.abs().max()
    return out, bound


def tolerance(out, bound, dtype):
    """The bound with the output's own rounding: half a step of its type relative to the value, and
    the smallest step's half near zero."""
    info = torch.finfo(dtype)
    return bound + (out.abs() + bound) * (info.eps / 2) + info.smallest_normal * info.eps


def quantise_cache(x: torch.Tensor):
    """A cache [N, Hkv, block, D] of 64-bit values as (e4m3 values in 64 bits, scales [N, Hkv])."""
    amax = x.abs().amax((2, 3))
    unit = torch.tensor([unit_of(a) for a in amax.flatten().tolist()], dtype=torch.float64).reshape(amax.shape)
    return nearest_e4m3(x / unit[:, :, None, None]), unit
