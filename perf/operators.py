"""Performance cases of the draft-scoring operators (hs_guard_b200.drafts): plain torch forms next to the calls.

A host model that drafts a tree of continuations has it scored before one branch is accepted. One tick of that path
is: positions and ancestor masks from the tree's parent links (``plan_tree``), norms and rotation of the queries and
keys (``norm_rope``), attention of the drafted tokens over each request's paged cache and their own ancestors
(``tree_attention``); then, for the accepted branch, pages and slots (``advance_tables``) and the copy of its keys and
values into the cache (``store_rows``). Each case is one of these operators at one size.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # a tick of the largest session bucket: every conversation accepts a few tokens, some roll back
        {"name": "tables tick", "op": "tables", "rows": 352, "page": 16, "len": 8000, "grow": 5},
        # many prompts admitted at once, with an odd page size
        {"name": "tables prompts", "op": "tables", "rows": 1000, "page": 48, "len": 2048, "grow": 2048},
        # one conversation, a small tree: latency
        {"name": "tree one", "op": "tree", "rows": 1, "nodes": 15, "len": 512, "chain": False},
        # a full server, wide trees
        {"name": "tree full", "op": "tree", "rows": 512, "nodes": 200, "len": 8000, "chain": False},
        # the classifier's attention layer (fp32 projection, q and gate interleaved, 64 of 256 dims rotated), one tree
        {"name": "norm one", "op": "norm", "tokens": 15, "hq": 8, "hkv": 2, "dim": 256, "rot": 64, "in": "fp32",
         "out": "fp16", "gate": True, "store": False, "len": 8000},
        # the same layer on a full server, keys and values going straight into the pages
        {"name": "norm full", "op": "norm", "tokens": 352 * 64, "hq": 8, "hkv": 2, "dim": 256, "rot": 64, "in": "fp32",
         "out": "fp16", "gate": True, "store": True, "len": 8000},
        # one conversation, one token, the classifier's window: latency
        {"name": "attend one", "op": "attend", "rows": 1, "nodes": 1, "hq": 8, "hkv": 2, "dim": 256, "len": 1000,
         "page": 16, "window": 512, "dtype": "fp16", "heads_first": False, "tree": False},
        # every slot of the headline server drafts a small tree, the classifier's window
        {"name": "attend slots", "op": "attend", "rows": 352, "nodes": 9, "hq": 8, "hkv": 2, "dim": 256, "len": 8000,
         "page": 16, "window": 512, "dtype": "fp16", "heads_first": False, "tree": True},
        # few long conversations without a window: the work is split along the cache
        {"name": "attend long", "op": "attend", "rows": 5, "nodes": 13, "hq": 32, "hkv": 8, "dim": 128, "len": 50001,
         "page": 64, "window": 0, "dtype": "bf16", "heads_first": True, "tree": True},
        # wide trees and many query heads for each key head: arithmetic counts as much as memory
        {"name": "attend wide", "op": "attend", "rows": 40, "nodes": 64, "hq": 32, "hkv": 4, "dim": 128, "len": 6000,
         "page": 32, "window": 0, "dtype": "bf16", "heads_first": False, "tree": True},
        # one accepted branch
        {"name": "store one", "op": "store", "tokens": 4, "hkv": 2, "dim": 256, "page": 16, "dtype": "fp16",
         "heads_first": False},
        # accepted branches and prompts of a full server
        {"name": "store full", "op": "store", "tokens": 30000, "hkv": 8, "dim": 128, "page": 64, "dtype": "bf16",
         "heads_first": True},
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["tables", "tree", "norm", "attend", "attend", "attend", "store"])
    if op == "tables":
        return {"op": op, "rows": _spread(rng, 1, 1000), "page": rng.choice([8, 16, 24, 32, 48, 64, 128]),
                "len": _spread(rng, 1, 8000), "grow": _spread(rng, 1, 2048)}
    if op == "tree":
        return {"op": op, "rows": _spread(rng, 1, 512), "nodes": _spread(rng, 1, 200), "len": _spread(rng, 1, 50000),
                "chain": rng.random() < 0.25}
    heads = rng.choice([(8, 2), (8, 8), (32, 8), (16, 2), (15, 5), (7, 1), (6, 2)])
    dim = rng.choice([64, 128, 256])
    if op == "norm":
        hq, hkv = heads
        top = max(1, 352 * 64 * 12 * 256 // ((hq + 2 * hkv) * dim))
        return {"op": op, "tokens": _spread(rng, 1, top), "hq": hq, "hkv": hkv, "dim": dim,
                "rot": rng.choice([dim, dim // 2, dim // 4]), "in": rng.choice(["fp32", "bf16", "fp16"]),
                "out": rng.choice(["fp16", "bf16"]), "gate": rng.random() < 0.5, "store": rng.random() < 0.5,
                "len": _spread(rng, 1, 50000)}
    dtype, heads_first = rng.choice(["fp16", "bf16"]), rng.random() < 0.5
    page = rng.choice([8, 16, 32, 48, 64, 128])
    if op == "store":
        return {"op": op, "tokens": _spread(rng, 1, 30000), "hkv": heads[1], "dim": dim, "page": page, "dtype": dtype,
                "heads_first": heads_first}
    while True:
        hq, hkv = rng.choice([(8, 2), (8, 8), (32, 8), (16, 2), (15, 5), (7, 1), (32, 4)])
        case = {"op": op, "rows": _spread(rng, 1, 352), "nodes": _spread(rng, 1, 64), "hq": hq, "hkv": hkv, "dim": dim,
                "len": _spread(rng, 1, 50000), "page": page, "window": rng.choice([0, 0, 512, _spread(rng, 3, 5000)]),
                "dtype": dtype, "heads_first": heads_first, "tree": rng.random() < 0.7}
        keys = case["rows"] * _reach(case)
        # no dearer than the largest listed cases: cache held, scores of the plain form
        if keys * hkv * dim <= 5 * 50001 * 8 * 128 and keys * hq * case["nodes"] <= 40 * 6000 * 32 * 64:
            return case


def _reach(case):
    """The most cached tokens a request of the case reads."""
    return min(case["len"], case["window"]) if case["window"] else case["len"]


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lengths(case, g):
    """Unequal lengths in [0, len]: most in the upper half, a few short, in a batch the first one full and one empty."""
    n, top = case["rows"], case["len"]
    u = torch.rand(n, generator=g, device="cuda")
    lens = (top * (0.5 + 0.5 * u)).to(torch.int32)
    lens = torch.where(torch.rand(n, generator=g, device="cuda") < 0.1, (top * u * u).to(torch.int32), lens)
    if n > 1:
        lens[0] = top
    if n > 2:
        lens[n // 2] = 0
    return lens


def _parents(counts, chain, g):
    """Parent links of `counts[b]` drafted tokens a request, parents first; -1 hangs on the last cached token. Trees as
    a drafter makes them: a few branches at each level, so the depth stays near the logarithm of the size."""
    total = int(counts.sum())
    cu = torch.zeros(len(counts) + 1, dtype=torch.int32, device="cuda")
    cu[1:] = torch.cumsum(counts, 0)
    index = torch.arange(total, device="cuda") - torch.repeat_interleave(cu[:-1].long(), counts.long())
    if chain:
        parents = index - 1
    else:
        u = torch.rand(total, generator=g, device="cuda")
        parents = torch.floor((index.float() * (0.35 + 0.3 * u))).long()
        parents = torch.where((index < 2) | (parents >= index), -1 * torch.ones_like(index), parents)
    return parents.to(torch.int32), cu


def _shares(n):
    """Numbers in [0, 1), evenly spread: which request has which is the seed's choice, their sum is the case's."""
    return (0.37 + 0.6180339887 * torch.arange(n, dtype=torch.float64, device="cuda")) % 1


def _counts(case, g):
    """Drafted tokens a request: half full, the others fewer; in a larger batch one request drafts nothing."""
    n, top = case["rows"], case["nodes"]
    c = torch.clamp(torch.floor(2 * top * _shares(n)), 1, top).to(torch.int32)
    c[0] = top
    if n > 3:
        c[3] = 0
    return c[torch.randperm(n, generator=g, device="cuda")]


def _pool(pages, page, hkv, dim, dtype, heads_first, g):
    """A cache [pages, page, hkv, dim], heads or tokens outermost within a page."""
    if heads_first:
        return torch.empty(pages, hkv, page, dim, dtype=dtype, device="cuda").normal_(generator=g).transpose(1, 2)
    return torch.empty(pages, page, hkv, dim, dtype=dtype, device="cuda").normal_(generator=g)


def _ancestors(parents, cu, words):
    """Ancestor bits [tokens, words] (int32), depths and requests; each round doubles how far up every token looks."""
    total = parents.shape[0]
    rows = torch.bucketize(torch.arange(total, device="cuda"), cu[1:], right=True)
    base = cu.long()[rows]
    up = torch.where(parents >= 0, base + parents, total)  # `total`: above the first drafted token
    up = torch.cat([up, up.new_full((1,), total)])
    bits = torch.zeros(total + 1, words * 32, dtype=torch.bool, device="cuda")
    bits[:total].scatter_(1, (torch.arange(total, device="cuda") - base)[:, None], True)
    for _ in range((words * 32).bit_length()):
        bits = bits | bits[up]
        up = up[up]
    bits = bits[:total]
    packed = (bits.view(total, words, 32) * (1 << torch.arange(32, device="cuda"))).sum(-1)
    packed = torch.where(packed >= 1 << 31, packed - (1 << 32), packed)
    return packed.to(torch.int32), bits.sum(-1) - 1, rows


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    s = {"case": case}
    if op == "tables":
        n, page = case["rows"], case["page"]
        lens = _lengths(case, g)
        who = torch.randperm(n, generator=g, device="cuda")
        delta = torch.floor((case["grow"] + 1) * _shares(n)).to(torch.int32)[who]
        back = who % 7 == 3  # rejected or finished: tokens taken back
        taken = (lens * torch.rand(n, generator=g, device="cuda")).to(torch.int32)
        delta = torch.where(back, -taken, delta)
        width = (case["len"] + case["grow"] + page - 1) // page
        held = (lens + page - 1) // page
        pages = n * width + 7
        # most of what the longest requests could want is free; sometimes not enough for the last ones
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        first = torch.cumsum(held, 0) - held
        column = torch.arange(width, device="cuda")
        table = torch.where(column < held[:, None], order[(first[:, None] + column).clamp(max=pages - 1)], -1)
        used = int(held.sum())
        want = int((((lens + delta.clamp(min=0) + page - 1) // page) - held).clamp(min=0).sum())
        free = max(1, min(pages - used, int(want * 0.97)))
        head = 5 * pages + 11  # a ring that has gone round several times
        ring = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        ring[(head + torch.arange(free, device="cuda")) % pages] = order[used:used + free]
        s.update(lens=lens, delta=delta, table=table.to(torch.int32).contiguous(), ring=ring, page=page,
                 counters=torch.tensor([head, head + free], dtype=torch.int64, device="cuda"),
                 capacity=int(delta.clamp(min=0).sum()) + 13)
    elif op == "tree":
        counts = _counts(case, g)
        parents, cu = _parents(counts, case["chain"], g)
        s.update(parents=parents, cu=cu, lens=_lengths(case, g), nodes=case["nodes"])
    elif op == "norm":
        t, hq, hkv, dim = case["tokens"], case["hq"], case["hkv"], case["dim"]
        step = 2 * dim if case["gate"] else dim  # q heads alone, or each followed by its gate
        width = hq * step + 2 * hkv * dim
        x = torch.empty(t, width, dtype=DTYPES[case["in"]], device="cuda").normal_(generator=g)
        out = DTYPES[case["out"]]
        s.update(q=x[:, :hq * step].view(t, hq, step)[:, :, :dim],
                 k=x[:, hq * step:hq * step + hkv * dim].view(t, hkv, dim),
                 v=x[:, hq * step + hkv * dim:].view(t, hkv, dim),
                 wq=1 + 0.2 * torch.randn(dim, generator=g, device="cuda"),
                 wk=1 + 0.2 * torch.randn(dim, generator=g, device="cuda"),
                 inv=10000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda").float() / case["rot"]),
                 positions=torch.randint(0, case["len"] + 1, (t,), generator=g, device="cuda").to(torch.int32),
                 eps=1e-6, out=out)
        if case["store"]:
            page = 16
            pages = (t + page - 1) // page + 3
            slots = torch.randperm(pages * page, generator=g, device="cuda")[:t].to(torch.int32)
            slots[t // 2] = -1  # a token that is not kept
            s.update(slots=slots, kc=torch.zeros(pages, page, hkv, dim, dtype=out, device="cuda"),
                     vc=torch.zeros(pages, page, hkv, dim, dtype=out, device="cuda"))
    elif op == "attend":
        hq, hkv, dim, page, dtype = case["hq"], case["hkv"], case["dim"], case["page"], DTYPES[case["dtype"]]
        lens, counts = _lengths(case, g), _counts(case, g)
        parents, cu = _parents(counts, not case["tree"], g)
        words = (case["nodes"] + 31) // 32
        mask, depth, rows = _ancestors(parents, cu, words)
        total = parents.shape[0]
        width = max(1, (case["len"] + page - 1) // page)
        first = (lens - case["window"] + 1).clamp(min=0) // page if case["window"] else torch.zeros_like(lens)
        last = (lens + page - 1) // page
        held = (last - first).clamp(min=0)  # pages before the window have been given back
        pages = int(held.sum()) + 2
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        column = torch.arange(width, device="cuda")
        at = torch.cumsum(held, 0)[:, None] - held[:, None] + column - first[:, None]
        kept = (column >= first[:, None]) & (column < last[:, None])
        table = torch.where(kept, order[at.clamp(0, pages - 1)], -1).to(torch.int32).contiguous()
        kc = _pool(pages, page, hkv, dim, dtype, case["heads_first"], g)
        vc = _pool(pages, page, hkv, dim, dtype, case["heads_first"], g)
        # memory that no token has filled yet: whatever was there, NaN among it
        junk = order[pages - 2:].long()
        kc[junk] = float("nan")
        vc[junk] = float("nan")
        part = (lens % page > 0) & (held > 0)
        ends = table.gather(1, (last - 1).clamp(min=0)[:, None].long())[:, 0].clamp(min=0).long()
        tail = part[:, None] & (torch.arange(page, device="cuda") >= (lens % page)[:, None])
        bad_page, bad_at = ends[:, None].expand_as(tail)[tail], torch.arange(page, device="cuda").expand_as(tail)[tail]
        kc[bad_page, bad_at] = float("nan")
        vc[bad_page, bad_at] = float("nan")
        s.update(q=torch.empty(total, hq, dim, dtype=dtype, device="cuda").normal_(generator=g),
                 k=torch.empty(total, hkv, dim, dtype=dtype, device="cuda").normal_(generator=g),
                 v=torch.empty(total, hkv, dim, dtype=dtype, device="cuda").normal_(generator=g),
                 kc=kc, vc=vc, table=table, lens=lens, cu=cu, mask=mask if case["tree"] else None,
                 positions=(lens[rows] + depth).to(torch.int32), scale=dim ** -0.5, window=case["window"],
                 nodes=case["nodes"])
    else:
        n, hkv, dim, page, dtype = case["tokens"], case["hkv"], case["dim"], case["page"], DTYPES[case["dtype"]]
        drafted = 2 * n + 3
        pages = (n + page - 1) // page + 2
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:n].to(torch.int32)
        if n > 2:
            slots[n // 3] = -1
        s.update(k=torch.empty(drafted, hkv, dim, dtype=dtype, device="cuda").normal_(generator=g),
                 v=torch.empty(drafted, hkv, dim, dtype=dtype, device="cuda").normal_(generator=g),
                 source=torch.randperm(drafted, generator=g, device="cuda")[:n].to(torch.int32), slots=slots,
                 kc=_pool(pages, page, hkv, dim, dtype, case["heads_first"], g),
                 vc=_pool(pages, page, hkv, dim, dtype, case["heads_first"], g))
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        from hs_guard_b200 import drafts
        if op == "tables":
            t = drafts.advance_tables(s["lens"], s["delta"], s["table"], s["ring"], s["counters"], s["page"],
                                      s["capacity"])
            return {"lens": t.lens, "counters": t.counters, "cu": t.cu, "slots": t.slots, "rows": t.rows,
                    "positions": t.positions, "table": s["table"], "ring": s["ring"]}
        if op == "tree":
            positions, mask = drafts.plan_tree(s["parents"], s["cu"], s["lens"], s["nodes"])
            return {"positions": positions, "mask": mask}
        if op == "norm":
            if "slots" in s:
                q = drafts.norm_rope_store(s["q"], s["k"], s["v"], s["wq"], s["wk"], s["inv"], s["positions"],
                                           s["eps"], s["kc"], s["vc"], s["slots"])
                return {"q": q, "k": s["kc"], "v": s["vc"]}
            q, k, v = drafts.norm_rope(s["q"], s["k"], s["v"], s["wq"], s["wk"], s["inv"], s["positions"], s["eps"],
                                       s["out"])
            return {"q": q, "k": k, "v": v}
        if op == "attend":
            out, lse = drafts.tree_attention(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["table"], s["lens"], s["cu"],
                                             s["scale"], max_tree=s["nodes"], mask=s["mask"],
                                             positions=s["positions"], window=s["window"])
            return {"out": out, "lse": lse}
        drafts.store_rows(s["k"], s["v"], s["kc"], s["vc"], s["slots"], s["source"])
        return {"k": s["kc"], "v": s["vc"]}
    return {"tables": _plain_tables, "tree": _plain_tree, "norm": _plain_norm, "attend": _plain_attend,
            "store": _plain_store}[op](s)


def _plain_tables(s):
    lens, page, table, ring, capacity = s["lens"].long(), s["page"], s["table"], s["ring"], s["capacity"]
    width, size = table.shape[1], ring.shape[0]
    head, tail = s["counters"][0], s["counters"][1]
    target = (lens + s["delta"]).clamp(min=0)
    target = torch.where(target > width * page, lens, target)
    before, after = (lens + page - 1) // page, (target + page - 1) // page
    need, back = (after - before).clamp(min=0), (before - after).clamp(min=0)
    upto = torch.cumsum(need, 0)
    served = (need == 0) | (upto <= tail - head)
    target = torch.where(served, target, lens)
    after = torch.where(served, after, before)
    taken = torch.where(served, need, 0)
    given = torch.cumsum(back, 0) - back
    column = torch.arange(width, device="cuda")
    fresh = (column >= before[:, None]) & (column < after[:, None])
    pick = (head + (upto - need)[:, None] + column - before[:, None]) % size
    freed = (column >= after[:, None]) & (column < before[:, None])
    where = (tail + given[:, None] + column - after[:, None]) % size
    ring[where[freed]] = table[freed]
    table.copy_(torch.where(fresh, ring[pick], table))
    grown = (target - lens).clamp(min=0)
    cu = torch.zeros(len(lens) + 1, dtype=torch.int64, device="cuda")
    cu[1:] = torch.cumsum(grown, 0)
    i = torch.arange(capacity, device="cuda")
    row = torch.searchsorted(cu[1:], i, right=True)
    live = i < cu[-1]
    row = torch.where(live, row, 0)
    position = lens[row] + i - cu[row]
    slot = table[row, (position // page).clamp(max=width - 1)] * page + position % page
    dead = torch.full_like(i, -1)
    return {"lens": target.to(torch.int32), "counters": torch.stack([head + taken.sum(), tail + back.sum()]),
            "cu": cu.to(torch.int32), "slots": torch.where(live, slot, dead).to(torch.int32),
            "rows": torch.where(live, row, dead).to(torch.int32),
            "positions": torch.where(live, position, dead).to(torch.int32), "table": table, "ring": ring}


def _plain_tree(s):
    mask, depth, rows = _ancestors(s["parents"], s["cu"], (s["nodes"] + 31) // 32)
    return {"positions": (s["lens"][rows] + depth).to(torch.int32), "mask": mask}


def _plain_norm(s):
    rot = s["inv"].shape[0]
    angle = s["positions"].float()[:, None] * s["inv"]
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]

    def one(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * w
        a, b = x[..., :rot], x[..., rot:2 * rot]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * rot:]], -1).to(s["out"])

    q, k, v = one(s["q"], s["wq"]), one(s["k"], s["wk"]), s["v"].to(s["out"])
    if "slots" not in s:
        return {"q": q, "k": k, "v": v}
    _put(s, k, v)
    return {"q": q, "k": s["kc"], "v": s["vc"]}


def _put(s, k, v):
    kept = s["slots"] >= 0
    slots, page = s["slots"][kept].long(), s["kc"].shape[1]
    s["kc"][slots // page, slots % page] = k[kept]
    s["vc"][slots // page, slots % page] = v[kept]


def _plain_store(s):
    at = s["source"].long()
    _put(s, s["k"][at], s["v"][at])
    return {"k": s["kc"], "v": s["vc"]}


def _plain_attend(s):
    case = s["case"]
    lens, cu, window, page = s["lens"].long(), s["cu"].long(), s["window"], case["page"]
    hq, hkv, dim, nodes, rows = case["hq"], case["hkv"], case["dim"], case["nodes"], case["rows"]
    reach = max(1, _reach(case))
    # the cached tokens a request can see, and its drafted ones, padded to the longest
    begin = (lens - window + 1).clamp(min=0) if window else torch.zeros_like(lens)
    kpos = begin[:, None] + torch.arange(reach, device="cuda")
    there = kpos < lens[:, None]
    at = torch.where(there, kpos, 0)
    page_of = s["table"].long().gather(1, at // page).clamp(min=0)
    node = torch.arange(nodes, device="cuda")
    drafted = node < (cu[1:] - cu[:-1])[:, None]
    token = torch.where(drafted, cu[:-1, None] + node, 0)

    def keys(pool, new):
        old = torch.where(there[..., None, None], pool[page_of, at % page].float(), 0.0)
        return torch.cat([old, torch.where(drafted[..., None, None], new[token].float(), 0.0)], 1).transpose(1, 2)

    q = s["q"][token].float().view(rows, nodes, hkv, hq // hkv, dim).permute(0, 2, 3, 1, 4)
    score = (q.reshape(rows, hkv, -1, dim) @ keys(s["kc"], s["k"]).transpose(-1, -2)) * s["scale"]
    score = score.view(rows, hkv, hq // hkv, nodes, reach + nodes)
    qpos = s["positions"].long()[token]
    see_old = there[:, None] & drafted[..., None]
    if s["mask"] is None:
        see_new = (node <= node[:, None])[None] & drafted[:, None] & drafted[..., None]
    else:
        bits = (s["mask"][token][..., None] >> torch.arange(32, device="cuda")) & 1
        see_new = (bits.view(rows, nodes, -1)[..., :nodes] != 0) & drafted[:, None] & drafted[..., None]
    if window:
        see_old = see_old & (kpos[:, None] > (qpos - window)[..., None])
        see_new = see_new & (qpos[:, None] > (qpos - window)[..., None])
    see = torch.cat([see_old, see_new], 2)[:, None, None]
    score = torch.where(see, score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = (p / torch.where(total > 0, total, 1.0)).view(rows, hkv, -1, reach + nodes) @ keys(s["vc"], s["v"])
    out = out.view(rows, hkv, hq // hkv, nodes, dim).permute(0, 3, 1, 2, 4).reshape(rows, nodes, hq, dim)
    lse = (top + torch.log(total))[..., 0].permute(0, 3, 1, 2).reshape(rows, nodes, hq)
    return {"out": out[drafted].to(s["q"].dtype), "lse": lse[drafted]}


# ---- 64-bit values --------------------------------------------------------------------------------------------------
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op in ("tables", "tree"):
        return None
    if op == "norm":
        inv, pos = s["inv"].double(), s["positions"].double()
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), pos[:, None, None] * inv)
        r = inv.shape[0]

        def one(x, w):
            x = x.double()
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + s["eps"]) * w.double()
            z = torch.complex(x[..., :r].contiguous(), x[..., r:2 * r].contiguous()) * turn
            return torch.cat([z.real, z.imag, x[..., 2 * r:]], -1)

        q, k, v = one(s["q"], s["wq"]), one(s["k"], s["wk"]), s["v"].double()
        if "slots" not in s:
            return {"q": q, "k": k, "v": v}
        kc, vc = s["kc"].double(), s["vc"].double()
        kept = (s["slots"] >= 0).nonzero()[:, 0]
        slots = s["slots"][kept].long()
        kc.view(-1, *kc.shape[2:])[slots] = k[kept]
        vc.view(-1, *vc.shape[2:])[slots] = v[kept]
        return {"q": q, "k": kc, "v": vc}
    if op == "store":
        kc, vc = s["kc"].double(), s["vc"].double()
        page = case["page"]
        for c, x in ((kc, s["k"]), (vc, s["v"])):
            kept = (s["slots"] >= 0).nonzero()[:, 0]
            slots = s["slots"][kept].long()
            c[torch.div(slots, page, rounding_mode="floor"), slots.remainder(page)] = x[s["source"][kept].long()].double()
        return {"k": kc, "v": vc}
    # request by request over the tokens it really has
    lens, cu = s["lens"].tolist(), s["cu"].tolist()
    group, page, window = case["hq"] // case["hkv"], case["page"], s["window"]
    outs, lses = [], []
    for b, length in enumerate(lens):
        a, z = cu[b], cu[b + 1]
        if z == a:
            continue
        start = max(0, length - window + 1) if window else 0
        at = torch.arange(start, length, device="cuda")
        where = s["table"][b][at // page].long()
        k = torch.cat([s["kc"][where, at % page], s["k"][a:z]]).double()
        v = torch.cat([s["vc"][where, at % page], s["v"][a:z]]).double()
        if s["mask"] is None:
            new = torch.ones(z - a, z - a, dtype=torch.bool, device="cuda").tril()
        else:
            j = torch.arange(z - a, device="cuda")
            new = (s["mask"][a:z][:, j // 32] >> (j % 32)) % 2 != 0
        see = torch.cat([torch.ones(z - a, len(at), dtype=torch.bool, device="cuda"), new], 1)
        if window:
            qp = s["positions"][a:z].long()
            see = see & (torch.cat([at, qp]) > qp[:, None] - window)
        score = torch.einsum("tghd,khd->hgtk", s["q"][a:z].double().unflatten(1, (case["hkv"], group)).transpose(1, 2),
                             k) * s["scale"]
        score = score.masked_fill(~see, float("-inf"))
        lse = torch.logsumexp(score, -1)
        weight = torch.exp(score - torch.where(lse == float("-inf"), torch.zeros_like(lse), lse)[..., None])
        out = torch.einsum("hgtk,khd->thgd", weight, v)
        outs.append(out.flatten(1, 2))
        lses.append(lse.permute(2, 0, 1).flatten(1, 2))
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}


# ---- work -----------------------------------------------------------------------------------------------------------
def work(case):
    """Bytes and operations of one pass, from the sizes alone: lengths and trees are 0.7 and 0.75 of their largest on
    average, the shares that prepare() gives them."""
    op = case["op"]
    if op == "tables":
        n, page = case["rows"], case["page"]
        tokens = n * case["grow"] * 0.85 / 2
        return {"bytes": n * 16 + tokens * 12 + 3 * 4 * tokens / page, "flops": 0}
    if op == "tree":
        nodes = case["rows"] * max(1, 0.75 * case["nodes"])
        return {"bytes": nodes * (8 + 4 * ((case["nodes"] + 31) // 32)) + 8 * case["rows"], "flops": 0}
    if op == "norm":
        t, e = case["tokens"], (case["hq"] + 2 * case["hkv"]) * case["dim"]
        return {"bytes": t * e * ((4 if case["in"] == "fp32" else 2) + 2) + 8 * t, "flops": 8 * t * e}
    if op == "store":
        return {"bytes": case["tokens"] * (2 * case["hkv"] * case["dim"] * 2 * 2 + 8), "flops": 0}
    b, one = case["rows"], case["rows"] == 1
    keys = b * max(1, min(case["len"] * (0.75 if one else 0.7), case["window"] or case["len"]))
    nodes = b * max(1, case["nodes"] * (1 if one else 0.75))
    moved = 2 * keys * case["hkv"] * case["dim"] * 2 + nodes * case["dim"] * 2 * (2 * case["hq"] + 2 * case["hkv"])
    return {"bytes": moved + nodes * 4 * case["hq"], "flops": 4 * keys / b * nodes * case["hq"] * case["dim"]}
