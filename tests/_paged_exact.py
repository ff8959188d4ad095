"""The paged attention in 64 bits on the GPU (for batches that the plain loops of _paged.py take too
long over), a bound on a kernel's error that has the weights' sum in it, the kernel's split of a batch
over its CTAs, and its parts of a weight."""

from __future__ import annotations

import torch

E4M3 = torch.float8_e4m3fn
WEIGHT_FLOOR = 2.0**-32  # half a step of the smallest weights, relative to the largest of a warp


def encode(x: torch.Tensor):
    """Values [N, Hkv, block, D] as the writer leaves them: e4m3 and power-of-two scales."""
    amax = x.abs().amax((2, 3)).double()
    m, e = torch.frexp(amax)
    e = torch.where(m <= 448 / 512, e - 9, e - 8)
    scale = torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, torch.full_like(e, -64)).clamp_min(-64))
    return (x.double() / scale[:, :, None, None]).float().to(E4M3), scale.float()


def rows(cache, scale, ids, n):
    """[Hkv, n, D] in 64 bits of the blocks `ids`."""
    x = cache.view(torch.uint8)[ids].view(E4M3).double() * scale[ids].double()[:, :, None, None]
    return x.transpose(0, 1).reshape(cache.shape[1], -1, cache.shape[3])[:, :n]


def attend(q, k, v, ks, vs, table, lens, cos, sin, skip=None):
    """(out, bound) [B, Hq, 1, D] in 64 bits. `skip` = (first, last): keys left out, for results that a
    test has to tell from the right one.

    Where the bound comes from, with p_j the softmax's weights:
    * a score is off by at most d_j = (2^-12 + 2^-14) sum_i |q_i k_ij| scale (query elements with 12
      significant bits, and the products' accumulation), a weight by the factor 1 + a_j, a_j = expm1(d_j);
    * the products use weights rounded to 11 bits, 2^-11, and the sums of products lose at most 2^-22 of
      sum_j |p_j v_j| at each of a fragment's n / 32 additions; 2^-16 is left for the exponentials and the
      factors of the warps and fragments;
    * weights end at an absolute WEIGHT_FLOOR of the largest p_j vs_j, times a value of at most 448;
    * the denominator is off by the factor 1 + sum_j p_j a_j, and 2^-16.
    """
    B, Hq, _, D = q.shape
    Hkv, block = k.shape[1], k.shape[2]
    G = Hq // Hkv
    out = torch.zeros(B, Hq, 1, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        ids = table[b, : -(-n // block)].long()
        c, s = cos[n - 1].double(), sin[n - 1].double()
        x, y = q[b, :, 0, : D // 2].double(), q[b, :, 0, D // 2 :].double()
        qr = torch.cat([x * c - y * s, y * c + x * s], -1).reshape(Hkv, G, D)
        kk, vv = rows(k, ks, ids, n), rows(v, vs, ids, n)
        unit = vs[ids].double().T.repeat_interleave(block, 1)[:, None, :n]
        if skip is not None:
            left = torch.ones(n, dtype=torch.bool, device=q.device)
            left[skip[0] : skip[1]] = False
            kk, vv, unit = kk[:, left], vv[:, left], unit[..., left]
        p = torch.softmax(qr @ kk.transpose(1, 2) * D**-0.5, -1)
        a = torch.expm1(qr.abs() @ kk.abs().transpose(1, 2) * (D**-0.5 * (2.0**-12 + 2.0**-14)))
        o = p @ vv
        sums = 2.0**-11 + 2.0**-16 + kk.shape[1] / 32 * 2.0**-22
        lost = kk.shape[1] * WEIGHT_FLOOR * 448 * (p * unit).amax(-1, keepdim=True)
        top = (p * (a + sums)) @ vv.abs() + lost
        low = (p * a).sum(-1, keepdim=True) + 2.0**-16
        out[b] = o.reshape(Hq, 1, D)
        bound[b] = ((top + o.abs() * low) / (1 - low)).reshape(Hq, 1, D)
    return out, bound


def tolerance(out, bound, dtype):
    """The bound and the output's own rounding, half a step, or half of its smallest one."""
    info = torch.finfo(dtype)
    return bound + (out.abs() + bound) * (info.eps / 2) + info.smallest_normal * info.eps


# ------------------------------------------------------------------------------ split over CTAs


def shape(Hq, Hkv, D):
    """(heads per unit, units per request, stages of K, charge of a unit's beginning, CTAs per SM)."""
    G = Hq // Hkv
    parts = (G + 7) // 8
    heads = -(-G // parts)
    hpu = 1 if heads <= 1 else 2 if heads <= 2 else 4 if heads <= 4 else 8
    return hpu, Hkv * parts, 4 if hpu == 8 else 3, 2 if D <= 128 else 1


def split(lens, Hq, Hkv, D, block, width, sms=148):
    """The kernel's fragments: a list per CTA of (unit, first chunk, end chunk, fragments of the unit),
    and whether whole pieces of units were taken."""
    _, ups, pen, per_sm = shape(Hq, Hkv, D)
    chunks = [max(1, -(-n // 128)) for n in lens]
    grid = min(sms * per_sm, 12 * 36, len(lens) * ups * -(-width * block // 128))
    ctas = [[] for _ in range(grid)]
    total = sum(chunks)
    if len(lens) * ups <= grid:
        per = -(-total * ups // grid)
        for x in range(per, per + 4):
            if sum(-(-c // x) for c in chunks) * ups <= grid:
                at = unit = 0
                for c in chunks:
                    k = -(-c // x)
                    for _ in range(ups):
                        q, r = divmod(c, k)
                        j = 0
                        for i in range(k):
                            e = j + q + (i < r)
                            ctas[at + i].append((unit, j, e, k))
                            j = e
                        at += k
                        unit += 1
                return ctas, True
    total = (total + len(lens) * pen) * ups
    per = -(-total // grid)
    base = unit = 0
    for c in chunks:
        for _ in range(ups):
            first, last = base + pen, base + pen + c  # positions of the unit's chunks
            nf = (last - 1) // per - first // per + 1
            for cta in range(first // per, (last - 1) // per + 1):
                lo, hi = max(first, cta * per), min(last, (cta + 1) * per)
                ctas[cta].append((unit, lo - first, hi - first, nf))
            base = last
            unit += 1
    return ctas, False


def parts_of_weight(x: torch.Tensor, steps=(5, 5, 5)):
    """The e4m3 parts of weights (64-bit tensor in [0, 256]) as the kernel takes them, and their sum."""
    r, f, total, parts = x.half().double(), 1.0, torch.zeros_like(x), []
    for k in (*steps, 0):
        e = r.float().clamp(max=448).to(E4M3).double()
        parts.append(e)
        total = total + e * f
        r, f = (r - e) * 2.0**k, f * 2.0**-k
    return parts, total

