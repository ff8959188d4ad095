"""Cases, inputs, plain forms and 64-bit results of the paged 8-bit KV cache operators.

Three operators of a generation loop over a paged cache held as e4m3 with one scale per
(block, KV head):

* ``tables``: block tables and slot maps from request lengths (``dominus_ultra_paged_tables``);
* ``write``: the new tokens' keys (rotated) and values quantised into their blocks
  (``dominus_ultra_paged_write``);
* ``attend``: single-token attention over the cache (``dominus_ultra_decode_paged``).

``own`` chooses between the plain torch forms and the framework's calls.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3_MAX = 448.0
SCALE_EXP_MIN = -64


def listed():
    return [
        # one short request, the latency of a call
        {"name": "attend one short", "op": "attend", "B": 1, "Hq": 8, "Hkv": 8, "D": 64, "L": 100, "even": True, "block": 16, "dtype": "bf16"},
        # one long request on a grouped-query layer: the sequence has to be split
        {"name": "attend one long", "op": "attend", "B": 1, "Hq": 32, "Hkv": 8, "D": 128, "L": 32768, "even": True, "block": 16, "dtype": "bf16"},
        # a serving batch of mixed lengths on a grouped-query layer
        {"name": "attend mixed batch", "op": "attend", "B": 64, "Hq": 32, "Hkv": 8, "D": 128, "L": 4096, "even": False, "block": 16, "dtype": "bf16"},
        # one key head for each query head
        {"name": "attend multi-head", "op": "attend", "B": 8, "Hq": 32, "Hkv": 32, "D": 64, "L": 2048, "even": True, "block": 32, "dtype": "fp16"},
        # groups of eight query heads, mixed lengths that end inside blocks
        {"name": "attend groups of 8", "op": "attend", "B": 16, "Hq": 64, "Hkv": 8, "D": 128, "L": 20001, "even": False, "block": 128, "dtype": "fp16"},
        # the long-context decode, the largest call
        {"name": "attend long context", "op": "attend", "B": 4, "Hq": 32, "Hkv": 8, "D": 128, "L": 131072, "even": True, "block": 64, "dtype": "bf16"},
        # one token of every request of a decode step
        {"name": "write one token each", "op": "write", "B": 64, "Hkv": 8, "D": 128, "T": 1, "past": 4095, "block": 16, "dtype": "bf16"},
        # a chunk of odd length behind blocks that are partly filled
        {"name": "write odd chunk", "op": "write", "B": 5, "Hkv": 32, "D": 64, "T": 777, "past": 1000, "block": 64, "dtype": "fp16"},
        # whole prompts of mixed lengths
        {"name": "write prompts", "op": "write", "B": 4, "Hkv": 8, "D": 128, "T": 8192, "past": 0, "block": 16, "dtype": "bf16"},
        # a decode step: one token for every request
        {"name": "tables of a step", "op": "tables", "B": 64, "T": 1, "cap": 8192, "block": 16, "kind": "step", "short": False},
        # prompts admitted together
        {"name": "tables of prompts", "op": "tables", "B": 16, "T": 4096, "cap": 16384, "block": 16, "kind": "prompts", "short": False},
        # a large batch in which requests end, begin and go on, with too few free blocks for all
        {"name": "tables of a turnover", "op": "tables", "B": 512, "T": 257, "cap": 8192, "block": 32, "kind": "turnover", "short": True},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "write", "tables"])
    block = rng.choice([16, 32, 64, 128])
    if op == "tables":
        B, T = _log_uniform(rng, 1, 1024), _log_uniform(rng, 1, 4096)
        T = max(1, min(T, (1 << 17) // B))
        cap = -(-(2 * T + _log_uniform(rng, 64, 8192)) // block) * block
        return {"op": op, "B": B, "T": T, "cap": cap, "block": block, "kind": rng.choice(["step", "prompts", "turnover"]), "short": rng.random() < 0.25}
    dtype = rng.choice(["bf16", "fp16"])
    Hq, Hkv, D = rng.choice([(8, 8, 64), (32, 32, 64), (32, 8, 128), (64, 8, 128), (32, 1, 64), (4, 2, 256), (12, 4, 32), (6, 2, 16)])
    if op == "write":
        B, T = _log_uniform(rng, 1, 128), _log_uniform(rng, 1, 8192)
        T = max(1, min(T, (1 << 25) // (B * Hkv * D)))
        return {"op": op, "B": B, "Hkv": Hkv, "D": D, "T": T, "past": rng.choice([0, rng.randint(1, 4096)]), "block": block, "dtype": dtype}
    B, L = _log_uniform(rng, 1, 128), _log_uniform(rng, 1, 131072)
    L = max(1, min(L, (1 << 29) // (B * Hkv * D)))
    return {"op": op, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "L": L, "even": rng.random() < 0.4, "block": block, "dtype": dtype}


# --------------------------------------------------------------------------------------- inputs


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=dtype)


def _randint(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device=DEVICE, dtype=torch.int32)


def _rope_tables(positions, D, dtype):
    # angles of far positions lose their fraction in 32 bits
    inv = 10000.0 ** (-torch.arange(0, D, 2, device=DEVICE, dtype=torch.float64) / D)
    a = torch.arange(positions, device=DEVICE, dtype=torch.float64)[:, None] * inv[None]
    return a.cos().to(dtype), a.sin().to(dtype)


def _filled_cache(g, blocks, Hkv, block, D):
    """A cache of unit-normal rows whose blocks and heads differ in size, as the writer leaves them."""
    x = _randn(g, blocks, Hkv, block, D, dtype=torch.float16)
    x = x * torch.exp2(_randint(g, -2, 3, blocks, Hkv, 1, 1).half())
    amax = x.abs().amax((2, 3)).float()
    m, e = torch.frexp(amax)
    e = torch.where(m <= E4M3_MAX / 512, e - 9, e - 8)
    scale = torch.ldexp(torch.ones_like(amax), e)
    x = (x / scale.half()[:, :, None, None]).to(torch.float8_e4m3fn)
    return x, scale


def _pages(tokens, block):
    return -(-tokens // block)


def _block_table(g, lens, block, width, blocks):
    """Rows of distinct scattered blocks, as many as each length needs; the rest -1."""
    need = (lens + block - 1) // block
    used = torch.arange(width, device=DEVICE)[None] < need[:, None]
    rank = (torch.cumsum(used.reshape(-1).int(), 0) - 1).reshape(used.shape)
    perm = torch.randperm(blocks, generator=g, device=DEVICE).int()
    return torch.where(used, perm[rank.clamp_min(0)], torch.full_like(rank, -1, dtype=torch.int32)), perm


def prepare(case, seed):
    g = _generator(seed)
    c = dict(case)
    if c["op"] == "attend":
        B, block, D, dt = c["B"], c["block"], c["D"], DTYPES[c["dtype"]]
        if c["even"]:
            lens = torch.full((B,), c["L"], device=DEVICE, dtype=torch.int32)
        else:
            lens = _randint(g, 1, c["L"] + 1, B)
            lens[0] = c["L"]
        width = _pages(c["L"], block)
        blocks = B * width + 3
        k, ks = _filled_cache(g, blocks, c["Hkv"], block, D)
        v, vs = _filled_cache(g, blocks, c["Hkv"], block, D)
        table, _ = _block_table(g, lens, block, width, blocks)
        cos, sin = _rope_tables(width * block, D, dt)
        # with the blocks' differing sizes a few keys stand out, as in trained heads
        q = _randn(g, B, c["Hq"], 1, D).to(dt)
        return {"case": c, "q": q, "k": k, "v": v, "ks": ks, "vs": vs, "table": table, "lens": lens, "cos": cos, "sin": sin}
    if c["op"] == "write":
        B, block, D, T, dt, Hkv = c["B"], c["block"], c["D"], c["T"], DTYPES[c["dtype"]], c["Hkv"]
        past = _randint(g, max(0, c["past"] - 37), c["past"] + 1, B)
        new = torch.full((B,), T, device=DEVICE, dtype=torch.int32)
        if T > 1:
            new = _randint(g, (T + 1) // 2, T + 1, B)
            new[0] = T
        # only the blocks that the call touches: the one that the past ends in, and new ones
        first = past // block
        width = _pages(T + block - 1, block) + 1
        blocks = B * width + 2
        k, ks = _filled_cache(g, blocks, Hkv, block, D)
        v, vs = _filled_cache(g, blocks, Hkv, block, D)
        ids = torch.randperm(blocks, generator=g, device=DEVICE)[: B * width].reshape(B, width)
        t = torch.arange(T, device=DEVICE)[None]
        pos = past[:, None].long() + t
        slots = torch.gather(ids, 1, pos // block - first[:, None].long()) * block + pos % block
        slots = torch.where(t < new[:, None], slots, torch.full_like(slots, -1)).int()
        size = torch.exp2(_randint(g, -1, 2, B, Hkv, 1, 1).float())
        kn = (_randn(g, B, Hkv, T, D) * size).to(dt)
        vn = (_randn(g, B, Hkv, T, D) * size).to(dt)
        cos, sin = _rope_tables(c["past"] + T, D, dt)
        return {"case": c, "kn": kn, "vn": vn, "k": k, "v": v, "ks": ks, "vs": vs, "slots": slots, "past": past, "cos": cos, "sin": sin}
    B, T, cap, block = c["B"], c["T"], c["cap"], c["block"]
    width = cap // block
    grow = _randint(g, (T + 1) // 2, T + 1, B)
    old = _randint(g, 1, cap - T + 1, B)
    if c["kind"] == "step":
        new = old + 1
    elif c["kind"] == "prompts":
        old = torch.where(_randint(g, 0, 4, B) == 0, old, torch.zeros_like(old))
        new = old + grow
    else:
        turn = _randint(g, 0, 4, B)
        old = torch.where(turn == 0, torch.zeros_like(old), old)
        new = torch.where(turn == 1, torch.zeros_like(old), torch.where(turn == 0, grow, old + 1))
        new = torch.where(turn == 3, (old - grow // 2).clamp_min(0), new)
    old_pages, new_pages = (old + block - 1) // block, (new + block - 1) // block
    need = int((new_pages - old_pages).clamp_min(0).sum())
    held = int(old_pages.sum())
    spare = need // 2 if c["short"] else need + 7
    blocks = B * width + 8  # what neither these requests hold nor is free belongs to others
    table, perm = _block_table(g, old, block, width, blocks)
    head = int(_randint(g, 0, blocks, 1)[0])
    ring = torch.full((blocks,), -1, device=DEVICE, dtype=torch.int32)
    ring[(head + torch.arange(spare, device=DEVICE)) % blocks] = perm[held : held + spare]
    state = torch.tensor([head, spare], device=DEVICE, dtype=torch.int32)
    return {"case": c, "table": table, "old": old.int(), "new": new.int(), "ring": ring, "state": state}


# ----------------------------------------------------------------------------------- plain forms


def _plain_attend(s):
    c = s["case"]
    B, Hq, Hkv, D, block = c["B"], c["Hq"], c["Hkv"], c["D"], c["block"]
    table = s["table"].clamp_min(0).long()
    keys = table.shape[1] * block

    def rows(cache, scale):
        x = cache.view(torch.uint8)[table].view(torch.float8_e4m3fn).float()  # [B, pages, Hkv, block, D]
        x = x * scale[table][:, :, :, None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, keys, D)

    at = (s["lens"].long() - 1).clamp_min(0)
    cos, sin = s["cos"][at].float()[:, None], s["sin"][at].float()[:, None]
    q = s["q"].float().reshape(B, Hq, D)
    q1, q2 = q[..., : D // 2], q[..., D // 2 :]
    q = torch.cat([q1 * cos - q2 * sin, q2 * cos + q1 * sin], -1).reshape(B, Hkv, Hq // Hkv, D)
    score = q @ rows(s["k"], s["ks"]).transpose(2, 3) / math.sqrt(D)
    seen = (torch.arange(keys, device=DEVICE)[None] < s["lens"][:, None])[:, None, None]
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = w.sum(-1, keepdim=True)
    v = rows(s["v"], s["vs"]).masked_fill(~seen[:, :, 0, :, None], 0.0)
    out = (w @ v) / torch.where(total > 0, total, torch.ones_like(total))
    return out.reshape(B, Hq, 1, D).to(s["q"].dtype)


def _to_e4m3(x):
    """64-bit values of at most 448 to the nearest e4m3 value, ties to even, rounded once."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 4).clamp_min(-9))
    return (torch.round(x / step) * step).float().to(torch.float8_e4m3fn)


def _plain_write_one(x, cache, scale, first, row0, count, blocks, block):
    """Rows x [B, Hkv, T, D] (64 bits) into the blocks [B, P] of one cache, in place."""
    B, Hkv, T, D = x.shape
    P = blocks.shape[1]
    t = (torch.arange(P * block, device=DEVICE)[None] - row0[:, None]).reshape(B, P, block)
    fresh = (t >= 0) & (t < count[:, None, None])
    old = (t < 0) & (count[:, None, None] > 0)
    at = t.clamp(0, T - 1).reshape(B, 1, P * block, 1).expand(B, Hkv, P * block, D)
    rows = torch.gather(x, 2, at).reshape(B, Hkv, P, block, D).transpose(1, 2)  # [B, P, Hkv, block, D]
    fresh5, old5 = fresh[:, :, None, :, None], old[:, :, None, :, None]
    amax = rows.abs().masked_fill(~fresh5, 0.0).amax((3, 4))
    m, e = torch.frexp(amax)
    e = torch.where(m <= E4M3_MAX / 512, e - 9, e - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, SCALE_EXP_MIN)).clamp_min(SCALE_EXP_MIN)
    want = torch.ldexp(torch.ones_like(amax), e)
    had = scale[blocks].double()
    held = old.any(2)[:, :, None]
    now = torch.where(held, torch.maximum(had, want), want)
    was = cache.view(torch.uint8)[blocks].view(torch.float8_e4m3fn)
    moved = was.double() * (had / now)[..., None, None]
    value = torch.where(fresh5, rows / now[..., None, None], torch.where(old5 & (now > had)[..., None, None], moved, torch.zeros_like(moved)))
    byte = _to_e4m3(value).view(torch.uint8)
    keep = ~fresh5 & ~(old5 & (now > had)[..., None, None])
    byte = torch.where(keep, was.view(torch.uint8), byte)
    touched = fresh.any(2)
    cache.view(torch.uint8)[blocks[touched]] = byte[touched]
    scale[blocks[touched]] = now[touched].float()


def _plain_write(s):
    c = s["case"]
    B, T, D, block = c["B"], c["T"], c["D"], c["block"]
    slots, past = s["slots"].long(), s["past"].long()
    count = (slots >= 0).sum(1)
    row0 = past % block
    P = _pages(T + block - 1, block)
    lead = (torch.arange(P, device=DEVICE)[None] * block - row0[:, None]).clamp_min(0)  # first new token of each page
    blocks = torch.gather(slots, 1, lead.clamp_max(T - 1)).clamp_min(0) // block
    at = (past[:, None] + torch.arange(T, device=DEVICE)[None]).clamp_max(s["cos"].shape[0] - 1)
    cos, sin = s["cos"][at].double()[:, None], s["sin"][at].double()[:, None]
    k1, k2 = s["kn"][..., : D // 2].double(), s["kn"][..., D // 2 :].double()
    k = torch.cat([k1 * cos - k2 * sin, k2 * cos + k1 * sin], -1)
    _plain_write_one(k, s["k"], s["ks"], past // block, row0, count, blocks, block)
    _plain_write_one(s["vn"].double(), s["v"], s["vs"], past // block, row0, count, blocks, block)
    return {"k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}


def _plain_tables(s):
    c = s["case"]
    B, T, block = c["B"], c["T"], c["block"]
    table, ring, state = s["table"], s["ring"], s["state"].long()
    width, N = table.shape[1], ring.shape[0]
    head, count = state[0], state[1]
    old, new = s["old"].long(), s["new"].long()
    op, np_ = (old + block - 1) // block, (new + block - 1) // block
    need = (np_ - op).clamp_min(0)
    served = (torch.cumsum(need, 0) <= count) | (need == 0)
    granted = torch.where(served, new, old)
    gp = torch.where(served, np_, op)
    page = torch.arange(width, device=DEVICE)[None]
    taken = (page >= op[:, None]) & (page < gp[:, None])
    freed = (page >= gp[:, None]) & (page < op[:, None])
    take_rank = torch.cumsum(taken.reshape(-1), 0).reshape(taken.shape) - 1
    free_rank = torch.cumsum(freed.reshape(-1), 0) - 1
    got = ring[((head + take_rank.clamp_min(0)) % N)]
    at = ((head + count + free_rank) % N)[freed.reshape(-1)]
    ring[at] = table[freed]
    table.copy_(torch.where(taken, got, table))
    pos = old[:, None] + torch.arange(T, device=DEVICE)[None]
    live = pos < granted[:, None]
    slot = torch.gather(table.long(), 1, (pos // block).clamp_max(width - 1)) * block + pos % block
    slots = torch.where(live, slot, torch.full_like(slot, -1)).int()
    out = torch.stack([(head + taken.sum()) % N, count - taken.sum() + freed.sum()]).int()
    return {"slots": slots, "lens": granted.int(), "state": out, "table": table, "ring": ring}


# ------------------------------------------------------------------------------------- one pass


def run(state):
    op = state["case"]["op"]
    if own:
        import dominusultra_b200 as du

        if op == "attend":
            return du.dominus_ultra_decode_paged(
                state["q"], state["k"], state["v"], state["ks"], state["vs"], state["table"], state["lens"], state["cos"], state["sin"]
            )
        if op == "write":
            du.dominus_ultra_paged_write(
                state["kn"], state["vn"], state["k"], state["v"], state["ks"], state["vs"], state["slots"], state["past"], state["cos"], state["sin"]
            )
            return {"k": state["k"], "v": state["v"], "ks": state["ks"], "vs": state["vs"]}
        slots, lens, left = du.dominus_ultra_paged_tables(
            state["table"], state["old"], state["new"], state["ring"], state["state"], state["case"]["block"], state["case"]["T"]
        )
        return {"slots": slots, "lens": lens, "state": left, "table": state["table"], "ring": state["ring"]}
    return {"attend": _plain_attend, "write": _plain_write, "tables": _plain_tables}[op](state)


def work(case):
    """Mean lengths stand for mixed ones: uniform over (0, L], or [T/2, T] new tokens."""
    c = case
    block = c["block"]
    if c["op"] == "attend":
        tokens = c["B"] * c["L"] if c["even"] else c["L"] + (c["B"] - 1) * (c["L"] + 1) / 2
        pages = tokens / block + (0 if c["even"] else c["B"] / 2)
        moved = 2 * tokens * c["Hkv"] * c["D"] + 8 * pages * c["Hkv"] + 4 * pages + 4 * c["B"]
        moved += 2 * 2 * c["B"] * c["Hq"] * c["D"] + 2 * 2 * c["B"] * (c["D"] // 2)
        return {"bytes": moved, "flops": 4 * tokens * c["Hq"] * c["D"]}
    if c["op"] == "write":
        tokens = c["T"] * c["B"] if c["T"] == 1 else c["T"] + (c["B"] - 1) * 0.75 * c["T"]
        pages = tokens / block + c["B"]
        moved = 2 * tokens * c["Hkv"] * c["D"] * (2 + 1) + 8 * pages * c["Hkv"] + 4 * c["B"] * (c["T"] + 1)
        moved += 2 * 2 * min(tokens, c["past"] + c["T"]) * (c["D"] // 2)
        return {"bytes": moved, "flops": 8 * tokens * c["Hkv"] * c["D"]}
    tokens = c["B"] if c["kind"] == "step" else 0.75 * c["B"] * c["T"]
    return {"bytes": 4 * (3 * c["B"] + c["B"] * c["T"] + 3 * tokens / block), "flops": c["B"] + tokens}


# ------------------------------------------------------------------------------------- 64 bits


def _exact_attend(s):
    c = s["case"]
    B, Hq, Hkv, D, block = c["B"], c["Hq"], c["Hkv"], c["D"], c["block"]
    G = Hq // Hkv
    out = torch.zeros(B, Hq, 1, D, device=DEVICE, dtype=torch.float64)
    for b, n in enumerate(s["lens"].tolist()):
        ids = s["table"][b, : _pages(n, block)].long()
        angle_cos, angle_sin = s["cos"][n - 1].double(), s["sin"][n - 1].double()
        q = s["q"][b, :, 0].double()
        turned = q.clone()
        turned[:, : D // 2] = q[:, : D // 2] * angle_cos - q[:, D // 2 :] * angle_sin
        turned[:, D // 2 :] = q[:, D // 2 :] * angle_cos + q[:, : D // 2] * angle_sin
        for h in range(Hkv):
            k = (s["k"][:, h].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double() * s["ks"][ids, h].double()[:, None, None]).reshape(-1, D)[:n]
            v = (s["v"][:, h].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double() * s["vs"][ids, h].double()[:, None, None]).reshape(-1, D)[:n]
            p = torch.softmax(turned[h * G : (h + 1) * G] @ k.T * D**-0.5, -1)
            out[b, h * G : (h + 1) * G, 0] = p @ v
    return out


def _nearest(x, grid):
    """The nearest of the sorted e4m3 values, a tie to the one with the even last bit."""
    hi = torch.searchsorted(grid, x.contiguous()).clamp(1, grid.numel() - 1)
    a, b = grid[hi - 1], grid[hi]
    pick_low = (x - a < b - x) | ((x - a == b - x) & ((hi - 1) % 2 == 0))
    return torch.where(pick_low, a, b)


def _exact_write(s):
    c = s["case"]
    D, block, T = c["D"], c["block"], c["T"]
    # magnitudes 0 .. 448 in the order of their bytes, so the index's parity is the last bit's
    grid = torch.arange(127, device=DEVICE, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    past, counts = s["past"].tolist(), (s["slots"] >= 0).sum(1).tolist()
    slots = s["slots"].tolist()
    k, v = s["k"].double(), s["v"].double()
    ks, vs = s["ks"].double(), s["vs"].double()
    cos, sin = s["cos"].double(), s["sin"].double()
    for b, n in enumerate(counts):
        p = torch.arange(past[b], past[b] + n, device=DEVICE)
        lo, hi = s["kn"][b, :, :n, : D // 2].double(), s["kn"][b, :, :n, D // 2 :].double()
        turned = torch.cat([lo * cos[p] - hi * sin[p], hi * cos[p] + lo * sin[p]], -1)
        for rows, cache, scale in ((turned, k, ks), (s["vn"][b, :, :n].double(), v, vs)):
            t = 0
            while t < n:
                blk, r = divmod(slots[b][t], block)
                m = min(n - t, block - r)
                part = rows[:, t : t + m]
                top = part.abs().amax((1, 2))
                unit = torch.full_like(top, 2.0**SCALE_EXP_MIN)
                e = torch.ceil(torch.log2(top.clamp_min(2.0**-100) / E4M3_MAX)).clamp_min(SCALE_EXP_MIN)
                for d in (-1, 0, 1):  # log2 may be a last bit off next to a power of two
                    unit = torch.where((torch.exp2(e - d) * E4M3_MAX >= top) & (e - d >= SCALE_EXP_MIN), torch.exp2(e - d), unit)
                if r > 0:
                    unit = torch.maximum(unit, scale[blk])
                    ratio = (scale[blk] / unit)[:, None, None]
                    back = cache[blk, :, :r] * ratio
                    cache[blk, :, :r] = torch.where(ratio < 1, _nearest(back.abs(), grid) * torch.sign(back), cache[blk, :, :r])
                x = part / unit[:, None, None]
                cache[blk, :, r : r + m] = _nearest(x.abs(), grid) * torch.sign(x)
                scale[blk] = unit
                t += m
    return {"k": k, "v": v, "ks": ks, "vs": vs}


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["B"] * _pages(case["T"], case["block"]) > 8192:
        return None  # block by block: over 20 seconds
    return _exact_write(s)
