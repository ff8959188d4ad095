"""Plain implementations of the operators on shared blocks, in Python integers, and of the attention of
several new tokens in 64 bits with a bound on a kernel's error."""

from __future__ import annotations

import torch

from tests import _paged_exact as exact

pages = lambda n, block: -(-n // block)  # noqa: E731


def fork(table, lens, sources, wanted, ring, state, block):
    """(table, copies, lengths, state) of a fork on lists; `ring` is updated in place."""
    B, width, N = len(table), len(table[0]), len(ring)
    cap = width * block
    head, count = state
    rows, kept = [], []
    for b in range(B):
        s, w = sources[b], wanted[b]
        own = 0 <= lens[b] <= cap
        ok = own and 0 <= s < B and 0 <= lens[s] <= cap and 0 <= w <= lens[s]
        kept.append(not ok)
        n = w if ok else (lens[b] if own else 0)
        rows.append((s if ok else b, n))
    before, after, whole, ends = set(), set(), set(), {}
    for b in range(B):
        if 0 <= lens[b] <= cap:
            before |= set(table[b][: pages(lens[b], block)])
        s, n = rows[b]
        held = table[s][: pages(n, block)]
        after |= set(held)
        if n % block and not kept[b]:
            ends.setdefault(held.pop(), []).append(b)
        whole |= set(held)
    inside = lambda ids: {x for x in ids if 0 <= x < N}  # noqa: E731
    freed = sorted(inside(before) - inside(after))
    if not (0 <= head < N and 0 <= count <= N) or count + len(freed) > N:
        return [list(r) for r in table], [[-1, -1] for _ in range(B)], list(lens), list(state)
    out, copies, lengths, taken = [], [], [], 0
    for b in range(B):
        s, n = rows[b]
        if kept[b]:
            out.append(list(table[b]))
            copies.append([-1, -1])
            lengths.append(lens[b])
            continue
        row, pair = table[s][: pages(n, block)], [-1, -1]
        if n % block and 0 <= row[-1] < N and (row[-1] in whole or min(ends[row[-1]]) != b):
            if taken < count:
                pair = [row[-1], ring[(head + taken) % N]]
                row = row[:-1] + [pair[1]]
                taken += 1
            else:
                row = row[:-1]
                n = len(row) * block
        out.append(row + [-1] * (width - len(row)))
        copies.append(pair)
        lengths.append(n)
    for i, x in enumerate(freed):
        ring[(head + count + i) % N] = x
    return out, copies, lengths, [(head + taken) % N, count - taken + len(freed)]


def compact(table, lens, ring, state, block):
    """(table, copies, ring, state) of a compaction on lists."""
    width, N = len(table[0]), len(ring)
    head, count = state
    held = [pages(n, block) if 0 <= n <= width * block else -1 for n in lens]
    used = {x for r, h in zip(table, held) if h > 0 for x in r[:h] if 0 <= x < N}
    free = [ring[(head + i) % N] for i in range(count)] if 0 <= head < N and 0 <= count <= N else [-1]
    if any(not 0 <= x < N for x in free) or len(set(free)) < len(free) or used & set(free):
        return [list(r) for r in table], [[-1, -1]] * (N // 2), list(ring), list(state)
    low = set(sorted(used | set(free))[: len(used)])
    moves = list(zip(sorted(used - low), sorted(low - used)))
    place = dict(moves)
    out = [list(r) if h < 0 else [place.get(x, x) for x in r[:h]] + [-1] * (width - h) for r, h in zip(table, held)]
    left = sorted((used | set(free)) - low)
    pairs = [list(m) for m in moves]
    return out, pairs + [[-1, -1]] * (N // 2 - len(pairs)), left + [-1] * (N - len(left)), [0, count]


def extend(q, k, v, ks, vs, table, past, lens, cos, sin):
    """(out, bound) [B, Hq, T, D] in 64 bits, on the tensors' device.

    The bound, with p_j the softmax's weights of a row:
    * query elements are carried as 16-bit values, 2^-11 of themselves and 2^-24 of the row's largest, and
      the products' accumulation takes 2^-14: a score is off by at most
      d_j = scale ((2^-11 + 2^-14) sum_i |q_i k_ij| + 2^-24 max_i |q_i| sum_i |k_ij|), a weight by the
      factor 1 + a_j, a_j = expm1(d_j);
    * the products use weights rounded to 11 bits, 2^-11, the sums of products lose at most 2^-22 of
      sum_j |p_j v_j| at each of a row's n / 16 additions, and 2^-16 is left for the exponentials and
      the factors that join the parts of a row;
    * weights end at an absolute 2^-32 of the largest p_j vs_j, times a value of at most 448;
    * the denominator is off by the factor 1 + sum_j p_j a_j, and 2^-16.

    The last step divides by 1 minus that sum, which only holds while the sum is below 1. From a half on
    (scores so large that a query's rounding changes the softmax) the bound is what holds for any
    weights: both results are means of the same values, so they are at most max v - min v <= 2 max |v|
    apart, times 1 + 2^-10 for the rounding of the weights and of the sums.
    """
    B, Hq, T, D = q.shape
    Hkv, block = k.shape[1], k.shape[2]
    G = Hq // Hkv
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b, (m, n) in enumerate(zip(past, lens)):
        t = n - m
        if t == 0:
            continue
        ids = table[b, : pages(n, block)].long()
        at = torch.arange(m, n, device=q.device)
        c, s = cos[at].double(), sin[at].double()
        x, y = q[b, :, :t, : D // 2].double(), q[b, :, :t, D // 2 :].double()
        qr = torch.cat([x * c - y * s, y * c + x * s], -1).reshape(Hkv, G * t, D)
        kk, vv = exact.rows(k, ks, ids, n), exact.rows(v, vs, ids, n)
        unit = vs[ids].double().T.repeat_interleave(block, 1)[:, None, :n]
        hidden = (torch.arange(n, device=q.device)[None] > at[:, None]).repeat(G, 1)[None]
        p = torch.softmax((qr @ kk.transpose(1, 2) * D**-0.5).masked_fill(hidden, -torch.inf), -1)
        off = qr.abs() @ kk.abs().transpose(1, 2) * (2.0**-11 + 2.0**-14)
        off += 2.0**-24 * qr.abs().amax(-1, keepdim=True) * kk.abs().sum(-1)[:, None]
        a = torch.expm1(D**-0.5 * off)
        o = p @ vv
        sums = 2.0**-11 + 2.0**-16 + n / 16 * 2.0**-22
        lost = n * 2.0**-32 * 448 * (p * unit).amax(-1, keepdim=True)
        top = (p * (a + sums)) @ vv.abs() + lost
        low = (p * a).sum(-1, keepdim=True) + 2.0**-16
        any_mean = (2 * (1 + 2.0**-10) * vv.abs().amax(1, keepdim=True)).expand_as(o)
        shape = (Hq, t, D)
        out[b, :, :t] = o.reshape(shape)
        bound[b, :, :t] = torch.where(low < 0.5, (top + o.abs() * low) / (1 - low), any_mean).reshape(shape)
    return out, bound


def make_cache(g, N, Hkv, block, D, device="cuda", spread=3):
    """A cache of unit-normal rows whose blocks differ in size by powers of two, on the device."""
    x = torch.randn(N, Hkv, block, D, generator=g) * torch.exp2(torch.randint(-spread, spread + 1, (N, Hkv, 1, 1), generator=g).double())
    c, s = exact.encode(x)
    return c.to(device), s.to(device)


def make_tables(g, lens, block, width, device="cuda"):
    """Scattered blocks for these lengths in a table of `width`, -1 behind; and the number of blocks."""
    need = [pages(n, block) for n in lens]
    N = sum(need) + 2
    order = torch.randperm(N, generator=g).tolist()
    rows = []
    for n in need:
        rows.append(order[:n] + [-1] * (width - n))
        order = order[n:]
    return torch.tensor(rows, dtype=torch.int32, device=device), N
