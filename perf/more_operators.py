"""Cases, inputs, plain forms and 64-bit results of the operators on a paged 8-bit KV cache that
several requests share, and of the attention of several new tokens over it.

Four operators of a serving loop:

* ``extend``: attention of a chunk of new tokens over the cache (``dominus_ultra_extend_paged``);
* ``fork``: requests that continue from others, or from a part of themselves
  (``dominus_ultra_paged_fork``);
* ``copy``: copies of blocks (``dominus_ultra_paged_copy``);
* ``compact``: blocks in use moved to the lowest ids (``dominus_ultra_paged_compact``).

``own`` chooses between the plain torch forms and the framework's calls.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3_MAX = 448.0
UNUSED = 2**31 - 1


def listed():
    return [
        # a draft of five tokens in one short request, the latency of a call
        {"name": "extend one short", "op": "extend", "B": 1, "Hq": 8, "Hkv": 8, "D": 64, "T": 5, "L": 100, "even": True, "block": 16, "dtype": "bf16"},
        # draft tokens of a serving batch of mixed lengths, to be accepted or not
        {"name": "extend drafts", "op": "extend", "B": 64, "Hq": 32, "Hkv": 8, "D": 128, "T": 4, "L": 4096, "even": False, "block": 16, "dtype": "bf16"},
        # more draft tokens behind long texts, groups of eight query heads
        {"name": "extend long drafts", "op": "extend", "B": 16, "Hq": 64, "Hkv": 8, "D": 128, "T": 16, "L": 20001, "even": False, "block": 128, "dtype": "fp16"},
        # prompts of odd lengths behind cached beginnings, one key head for each query head
        {"name": "extend mixed prompts", "op": "extend", "B": 8, "Hq": 32, "Hkv": 32, "D": 64, "T": 777, "L": 2048, "even": False, "block": 32, "dtype": "fp16"},
        # a question behind a long text
        {"name": "extend a long text", "op": "extend", "B": 1, "Hq": 32, "Hkv": 8, "D": 128, "T": 256, "L": 32768, "even": True, "block": 16, "dtype": "bf16"},
        # the last chunk of a long prompt, the largest call
        {"name": "extend by a large chunk", "op": "extend", "B": 1, "Hq": 32, "Hkv": 8, "D": 128, "T": 2048, "L": 32768, "even": True, "block": 64, "dtype": "bf16"},
        # a step of a beam search: 16 searches of four beams each
        {"name": "fork beams", "op": "fork", "B": 64, "cap": 4096, "block": 16, "kind": "beams", "short": False},
        # a large batch in which requests end, shrink, or begin with a part of another's text, with too few free blocks for all
        {"name": "fork prefixes", "op": "fork", "B": 512, "cap": 8192, "block": 32, "kind": "prefixes", "short": True},
        # the partly filled blocks of a beam search's step, some beams without one
        {"name": "copy a step's blocks", "op": "copy", "n": 64, "Hkv": 8, "D": 128, "block": 16, "used": 0.5},
        # the moves of a compaction
        {"name": "copy a compaction's blocks", "op": "copy", "n": 4096, "Hkv": 8, "D": 128, "block": 32, "used": 0.9},
        # a small cache with holes
        {"name": "compact a small cache", "op": "compact", "B": 16, "cap": 4096, "block": 64, "full": 0.5},
        # a large cache after many requests have gone
        {"name": "compact a large cache", "op": "compact", "B": 256, "cap": 8192, "block": 16, "full": 0.6},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["extend", "extend", "extend", "fork", "copy", "compact"])
    block = rng.choice([16, 32, 64, 128])
    if op == "fork":
        B = _log_uniform(rng, 1, 512)
        cap = _log_uniform(rng, 1, min(512, (1 << 17) // B)) * block
        return {"op": op, "B": B, "cap": cap, "block": block, "kind": rng.choice(["beams", "prefixes"]), "short": rng.random() < 0.25}
    if op == "compact":
        B = _log_uniform(rng, 1, 256)
        cap = _log_uniform(rng, 1, min(512, (1 << 17) // B)) * block
        return {"op": op, "B": B, "cap": cap, "block": block, "full": rng.uniform(0.05, 0.95)}
    Hq, Hkv, D = rng.choice([(8, 8, 64), (32, 32, 64), (32, 8, 128), (64, 8, 128), (32, 1, 64), (4, 2, 256), (12, 4, 32), (6, 2, 16)])
    if op == "copy":
        n = max(1, min(_log_uniform(rng, 1, 4096), (1 << 27) // (Hkv * block * D)))
        return {"op": op, "n": n, "Hkv": Hkv, "D": D, "block": block, "used": rng.uniform(0.2, 1.0)}
    dtype = rng.choice(["bf16", "fp16"])
    B, T, L = _log_uniform(rng, 1, 128), _log_uniform(rng, 1, 2048), _log_uniform(rng, 1, 32768)
    T = max(1, min(T, (1 << 26) // (B * Hq * D)))  # the queries
    L = max(1, min(L, (1 << 28) // (B * Hkv * D), (1 << 38) // (B * Hq * T * max(D, 128))))  # the cache; the products
    return {"op": op, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "T": min(T, L), "L": L, "even": rng.random() < 0.4, "block": block, "dtype": dtype}


# --------------------------------------------------------------------------------------- inputs


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=dtype)


def _randint(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device=DEVICE, dtype=torch.int32)


def _pages(tokens, block):
    return (tokens + block - 1) // block


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
    return (x / scale.half()[:, :, None, None]).to(torch.float8_e4m3fn), scale


def _block_table(g, pages, width, blocks):
    """Rows of distinct scattered blocks, `pages` of them in each row, then -1; and the order that
    they were taken in, from which the first sum(pages) are used."""
    used = torch.arange(width, device=DEVICE)[None] < pages[:, None]
    rank = (torch.cumsum(used.reshape(-1), 0) - 1).reshape(used.shape)
    order = torch.randperm(blocks, generator=g, device=DEVICE).int()
    return torch.where(used, order[rank.clamp_min(0)], torch.full_like(order[:1], -1)), order


def _ring(g, order, held, spare, blocks):
    """A ring of free blocks that begins anywhere: the `spare` ones behind the `held` ones of the order."""
    head = int(_randint(g, 0, blocks, 1)[0])
    ring = torch.full((blocks,), -1, device=DEVICE, dtype=torch.int32)
    ring[(head + torch.arange(spare, device=DEVICE)) % blocks] = order[held : held + spare]
    return ring, torch.tensor([head, spare], device=DEVICE, dtype=torch.int32)


def prepare(case, seed):
    g = _generator(seed)
    c = dict(case)
    block = c["block"]
    if c["op"] == "extend":
        B, D, T, L, dt = c["B"], c["D"], c["T"], c["L"], DTYPES[c["dtype"]]
        new = torch.full((B,), T, device=DEVICE, dtype=torch.int32)
        lens = torch.full((B,), L, device=DEVICE, dtype=torch.int32)
        if not c["even"]:
            new[1:] = _randint(g, (T + 1) // 2, T + 1, B - 1)
            lens[1:] = _randint(g, T, L + 1, B - 1)
        width = _pages(L, block)
        blocks = B * width + 3
        k, ks = _filled_cache(g, blocks, c["Hkv"], block, D)
        v, vs = _filled_cache(g, blocks, c["Hkv"], block, D)
        table, _ = _block_table(g, _pages(lens, block), width, blocks)
        cos, sin = _rope_tables(width * block, D, dt)
        # with the blocks' differing sizes a few keys stand out, as in trained heads
        q = _randn(g, B, c["Hq"], T, D).to(dt)
        return {"case": c, "q": q, "k": k, "v": v, "ks": ks, "vs": vs, "table": table, "past": lens - new, "lens": lens, "cos": cos, "sin": sin}
    if c["op"] == "copy":
        n = c["n"]
        blocks = 2 * n + 5
        k, ks = _filled_cache(g, blocks, c["Hkv"], block, c["D"])
        v, vs = _filled_cache(g, blocks, c["Hkv"], block, c["D"])
        pairs = torch.randperm(blocks, generator=g, device=DEVICE)[: 2 * n].reshape(n, 2).int()
        gone = torch.rand(n, 1, generator=g, device=DEVICE) > c["used"]
        gone[0] = False
        return {"case": c, "k": k, "v": v, "ks": ks, "vs": vs, "copies": torch.where(gone, torch.full_like(pairs, -1), pairs)}
    B, cap = c["B"], c["cap"]
    width = cap // block
    if c["op"] == "compact":
        lo, hi = max(0, int((2 * c["full"] - 1) * cap)), min(cap, int(2 * c["full"] * cap))
        lens = _randint(g, lo, hi + 1, B)
        pages = _pages(lens, block)
        held = int(pages.sum())
        blocks = B * width + 3
        table, order = _block_table(g, pages, width, blocks)
        # most of what these requests do not hold is free, some belongs to others
        spare = (blocks - held) * 15 // 16
        ring, state = _ring(g, order, held, spare, blocks)
        return {"case": c, "table": table, "lens": lens, "ring": ring, "state": state}
    row = torch.arange(B, device=DEVICE, dtype=torch.int32)
    blocks = B * width + 8
    if c["kind"] == "beams":
        first = row - row % 4
        lens = _randint(g, 1, cap + 1, B)[first]
        source = torch.minimum(first + _randint(g, 0, 4, B), torch.full_like(row, B - 1))
        wanted = lens
    else:
        first = torch.where(_randint(g, 0, 3, B) == 0, torch.zeros_like(row), row)
        lens = _randint(g, 0, cap + 1, B)
        turn = _randint(g, 0, 4, B)
        source = torch.where(turn == 0, _randint(g, 0, B, B), row)
        part = (torch.rand(B, generator=g, device=DEVICE) * (lens[source] + 1)).int().clamp_max(lens[source])
        wanted = torch.where(turn == 1, torch.zeros_like(row), torch.where(turn == 3, lens, part))
    # a beginning of whole blocks that rows share with another
    whole = torch.minimum(lens, lens[first]) // block
    common = (torch.rand(B, generator=g, device=DEVICE) * (whole + 1)).int().clamp_max(whole)
    common = torch.where(first == row, torch.zeros_like(common), common)
    pages = _pages(lens, block)
    own_pages = pages - common
    table, order = _block_table(g, own_pages, width, blocks)
    page = torch.arange(width, device=DEVICE)[None]
    shifted = torch.gather(table, 1, (page - common[:, None]).clamp_min(0).long())
    table = torch.where(page < common[:, None], table[first], shifted)
    table = torch.where(page < pages[:, None], table, torch.full_like(table, -1))
    held = int(own_pages.sum())
    ring, state = _ring(g, order, held, min(B // 16 if c["short"] else B + 3, blocks - held), blocks)
    return {"case": c, "table": table, "lens": lens, "sources": source, "wanted": wanted, "ring": ring, "state": state}


# ----------------------------------------------------------------------------------- plain forms


def _plain_extend(s):
    c = s["case"]
    B, Hq, Hkv, D, T, block = c["B"], c["Hq"], c["Hkv"], c["D"], c["T"], c["block"]
    G = Hq // Hkv
    table = s["table"].clamp_min(0).long()
    keys = table.shape[1] * block

    def rows(cache, scale):
        x = cache.view(torch.uint8)[table].view(torch.float8_e4m3fn).float()  # [B, pages, Hkv, block, D]
        x = x * scale[table][:, :, :, None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, keys, D)

    past, lens = s["past"].long(), s["lens"].long()
    at = past[:, None] + torch.arange(T, device=DEVICE)[None]  # [B, T], the query's position
    live = at < lens[:, None]
    cos = s["cos"][at.clamp_max(s["cos"].shape[0] - 1)].float()[:, None]
    sin = s["sin"][at.clamp_max(s["sin"].shape[0] - 1)].float()[:, None]
    q1, q2 = s["q"][..., : D // 2].float(), s["q"][..., D // 2 :].float()
    q = torch.cat([q1 * cos - q2 * sin, q2 * cos + q1 * sin], -1).reshape(B, Hkv, G * T, D)
    score = (q @ rows(s["k"], s["ks"]).transpose(2, 3) / math.sqrt(D)).reshape(B, Hkv, G, T, keys)
    key = torch.arange(keys, device=DEVICE)
    seen = (key[None, None] <= at[:, :, None]) & live[:, :, None]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    w = score.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    total = w.sum(-1, keepdim=True)
    v = rows(s["v"], s["vs"]).masked_fill((key[None] >= lens[:, None])[:, None, :, None], 0.0)
    out = (w.reshape(B, Hkv, G * T, keys) @ v).reshape(B, Hkv, G, T, D)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    return out.reshape(B, Hq, T, D).to(s["q"].dtype)


def _plain_fork(s):
    block = s["case"]["block"]
    old_table, ring = s["table"].long(), s["ring"]
    B, width = old_table.shape
    N = ring.shape[0]
    head, count = s["state"][0].long(), s["state"][1].long()
    new = s["wanted"].long()
    b = torch.arange(B, device=DEVICE)
    page = torch.arange(width, device=DEVICE)[None]
    rows = old_table[s["sources"].long()]
    pages = _pages(new, block)
    held = page < pages[:, None]
    partly = (new % block != 0)[:, None] & (page == pages[:, None] - 1)
    # the lowest claim to each block: 0 for one that holds it whole, else the request's number
    claim = torch.where(partly, b[:, None] + 1, torch.zeros_like(rows))
    where = torch.where(held, rows, torch.full_like(rows, N))
    owner = torch.full((N + 1,), UNUSED, device=DEVICE, dtype=torch.long)
    owner = owner.scatter_reduce(0, where.reshape(-1), claim.reshape(-1), "amin")[:N]
    last = torch.gather(rows, 1, (pages[:, None] - 1).clamp_min(0))[:, 0]
    need = partly.any(1) & (owner[last.clamp_min(0)] != b + 1)
    rank = torch.cumsum(need, 0)
    served = need & (rank <= count)
    cut = need & ~served
    pages = torch.where(cut, pages - 1, pages)
    new = torch.where(cut, pages * block, new)
    got = ring[(head + (rank - 1).clamp_min(0)) % N].long()
    table = torch.where(partly & served[:, None], got[:, None], rows)
    table = torch.where(page < pages[:, None], table, torch.full_like(table, -1))
    copies = torch.where(served[:, None], torch.stack([last, got], 1), torch.full((B, 2), -1, device=DEVICE))
    had = torch.zeros(N + 1, device=DEVICE, dtype=torch.long)
    had = had.scatter(0, torch.where(page < _pages(s["lens"].long(), block)[:, None], old_table, torch.full_like(rows, N)).reshape(-1), 1)[:N]
    freed = (had > 0) & (owner == UNUSED)
    to = (head + count + torch.cumsum(freed, 0) - 1) % N
    ring[to[freed]] = torch.arange(N, device=DEVICE, dtype=torch.int32)[freed]
    taken = served.sum()
    state = torch.stack([(head + taken) % N, count - taken + freed.sum()]).int()
    return {"table": table.int(), "copies": copies.int(), "lens": new.int(), "state": state, "ring": ring}


def _plain_copy(s):
    src, dst = s["copies"].long().unbind(1)
    keep = src >= 0
    src, dst = src[keep], dst[keep]
    k, v = s["k"].view(torch.uint8), s["v"].view(torch.uint8)
    k[dst], v[dst] = k[src], v[src]
    s["ks"][dst], s["vs"][dst] = s["ks"][src], s["vs"][src]
    return {"k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}


def _plain_compact(s):
    block = s["case"]["block"]
    table, ring = s["table"].long(), s["ring"].long()
    N, width = ring.shape[0], table.shape[1]
    head, count = s["state"][0].long(), s["state"][1].long()
    ids = torch.arange(N, device=DEVICE)
    held = torch.arange(width, device=DEVICE)[None] < _pages(s["lens"].long(), block)[:, None]
    none = torch.full_like(table, N)
    used = torch.zeros(N + 1, device=DEVICE, dtype=torch.bool).scatter(0, torch.where(held, table, none).reshape(-1), True)[:N]
    at = (ids - head) % N  # each entry's place behind the ring's head
    free = torch.zeros(N + 1, device=DEVICE, dtype=torch.bool).scatter(0, torch.where(at < count, ring, torch.full_like(ring, N)), True)[:N]
    ours = used | free
    low = ours & (torch.cumsum(ours, 0) <= used.sum())
    beyond = torch.full_like(ids, N)
    movers = torch.sort(torch.where(used & ~low, ids, beyond))[0]
    holes = torch.sort(torch.where(free & low, ids, beyond))[0]
    moves = movers < N
    copies = torch.where(moves[:, None], torch.stack([movers, holes], 1), torch.full((N, 2), -1, device=DEVICE))[: N // 2]
    place = torch.cat([ids, beyond[:1]]).scatter(0, movers, holes)
    rows = torch.where(held, place[table.clamp_min(0)], torch.full_like(table, -1))
    left = torch.sort(torch.where(ours & ~low, ids, beyond))[0]
    ring = torch.where(left < N, left, torch.full_like(left, -1))
    return {"table": rows.int(), "copies": copies.int(), "ring": ring.int(), "state": torch.stack([torch.zeros_like(count), count]).int()}


# ------------------------------------------------------------------------------------- one pass


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        import dominusultra_b200 as du

        if op == "extend":
            return du.dominus_ultra_extend_paged(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["table"], s["past"], s["lens"], s["cos"], s["sin"])
        if op == "fork":
            table, copies, lens, left = du.dominus_ultra_paged_fork(
                s["table"], s["lens"], s["sources"], s["wanted"], s["ring"], s["state"], s["case"]["block"]
            )
            return {"table": table, "copies": copies, "lens": lens, "state": left, "ring": s["ring"]}
        if op == "copy":
            du.dominus_ultra_paged_copy(s["k"], s["v"], s["ks"], s["vs"], s["copies"])
            return {"k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}
        table, copies, ring, left = du.dominus_ultra_paged_compact(s["table"], s["lens"], s["ring"], s["state"], s["case"]["block"])
        return {"table": table, "copies": copies, "ring": ring, "state": left}
    return {"extend": _plain_extend, "fork": _plain_fork, "copy": _plain_copy, "compact": _plain_compact}[op](s)


def work(case):
    """Mean lengths stand for mixed ones."""
    c = case
    block = c["block"]
    if c["op"] == "extend":
        B, T, L = c["B"], c["T"], c["L"]
        others = 0 if c["even"] else B - 1
        new = (B - others) * T + others * 0.75 * T
        tokens = (B - others) * L + others * (T + L) / 2
        pairs = (B - others) * T * (L - T / 2) + others * 0.75 * T * ((T + L) / 2 - 0.375 * T)
        moved = 2 * tokens * c["Hkv"] * c["D"] + (8 * c["Hkv"] + 4) * (tokens / block + others / 2) + 8 * B
        moved += 2 * 2 * new * c["Hq"] * c["D"] + 2 * 2 * new * (c["D"] // 2)
        return {"bytes": moved, "flops": 4 * pairs * c["Hq"] * c["D"]}
    if c["op"] == "copy":
        pairs = max(1, c["n"] * c["used"])
        return {"bytes": 2 * pairs * (2 * c["Hkv"] * block * c["D"] + 8 * c["Hkv"]) + 8 * c["n"], "flops": 0}
    entries = c["B"] * (c["cap"] / block)
    if c["op"] == "fork":
        return {"bytes": 4 * (0.5 * entries + entries + 6 * c["B"]), "flops": entries}
    return {"bytes": 4 * (c["full"] * entries + entries + 2 * entries + c["B"]), "flops": 2 * entries}


# ------------------------------------------------------------------------------------- 64 bits


def _exact_extend(s):
    c = s["case"]
    B, Hq, Hkv, D, T, block = c["B"], c["Hq"], c["Hkv"], c["D"], c["T"], c["block"]
    G = Hq // Hkv
    out = torch.zeros(B, Hq, T, D, device=DEVICE, dtype=torch.float64)
    past, lens = s["past"].tolist(), s["lens"].tolist()
    half = D // 2
    for b in range(B):
        n, new = lens[b], lens[b] - past[b]
        if not new:
            continue
        ids = s["table"][b, : _pages(n, block)].long()
        where = torch.arange(past[b], n, device=DEVICE)
        cos, sin = s["cos"][where].double(), s["sin"][where].double()
        hidden = torch.arange(n, device=DEVICE)[None] > where[:, None]
        for h in range(Hkv):
            k = (s["k"][:, h].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double() * s["ks"][ids, h].double()[:, None, None]).reshape(-1, D)[:n]
            v = (s["v"][:, h].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double() * s["vs"][ids, h].double()[:, None, None]).reshape(-1, D)[:n]
            for i in range(h * G, (h + 1) * G):
                q = s["q"][b, i, :new].double()
                turned = torch.empty_like(q)
                turned[:, :half] = q[:, :half] * cos - q[:, half:] * sin
                turned[:, half:] = q[:, half:] * cos + q[:, :half] * sin
                p = torch.softmax((turned @ k.T * D**-0.5).masked_fill(hidden, -math.inf), -1)
                out[b, i, :new] = p @ v
    return out


def exact(case, seed):
    if case["op"] in ("fork", "compact"):
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "extend":
        return _exact_extend(s)
    k, v, ks, vs = s["k"].double(), s["v"].double(), s["ks"].double(), s["vs"].double()
    for src, dst in s["copies"].tolist():
        if src >= 0:
            for x in (k, v, ks, vs):
                x[dst] = x[src]
    return {"k": k, "v": v, "ks": ks, "vs": vs}
