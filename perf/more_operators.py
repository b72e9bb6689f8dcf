"""Performance cases of the 8-bit cache and of token log-probabilities (hs_guard_b200.drafts): plain torch forms next to the calls.

A host model whose keys and values are kept in 8 bits (e4m3, a scale for each block of tokens and key head) makes three
calls a tick beside its projections: ``append_8bit`` rotates queries and keys and writes keys and values into the pages,
``attention_8bit`` lets the newest tokens of each request (one, a drafted tree or a chunk of a prompt) attend what their
pages hold, and ``token_logprobs`` says from the logits how likely the drafted tokens were and what else could have come.
Each case is one of these operators at one size.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
F8 = torch.float8_e4m3fn


def listed():
    return [
        # one conversation generates a token, the classifier's attention layout (64 of 256 dims rotated): latency
        {"name": "append one", "op": "append", "rows": 1, "grow": 1, "hq": 8, "hkv": 2, "dim": 256, "rot": 64, "len": 8000,
         "page": 16, "block": 16, "pairs": False, "factor": 1.0, "dtype": "fp16", "heads_first": False},
        # every slot of the headline server appends a few tokens, interleaved rotation stretched for long contexts
        {"name": "append slots", "op": "append", "rows": 352, "grow": 5, "hq": 32, "hkv": 8, "dim": 128, "rot": 128, "len": 8000,
         "page": 64, "block": 32, "pairs": True, "factor": 1.2079, "dtype": "bf16", "heads_first": True},
        # prompts admitted at once
        {"name": "append prompts", "op": "append", "rows": 20, "grow": 2500, "hq": 32, "hkv": 8, "dim": 128, "rot": 128,
         "len": 2000, "page": 64, "block": 64, "pairs": False, "factor": 1.0, "dtype": "bf16", "heads_first": False},
        # one conversation, one token, the classifier's window and four first tokens that stay visible: latency
        {"name": "attend one", "op": "attend", "rows": 1, "nodes": 1, "hq": 8, "hkv": 2, "dim": 256, "len": 8000, "page": 16,
         "block": 16, "window": 512, "sinks": 4, "dtype": "fp16", "heads_first": False, "tree": False},
        # every slot of the headline server, one or two tokens each, the same window
        {"name": "attend slots", "op": "attend", "rows": 352, "nodes": 2, "hq": 8, "hkv": 2, "dim": 256, "len": 8000, "page": 16,
         "block": 16, "window": 512, "sinks": 4, "dtype": "fp16", "heads_first": False, "tree": False},
        # a batch of short conversations, a key head for every query head, pages of 8 tokens
        {"name": "attend steps", "op": "attend", "rows": 64, "nodes": 1, "hq": 16, "hkv": 16, "dim": 64, "len": 2100, "page": 8,
         "block": 8, "window": 0, "sinks": 0, "dtype": "bf16", "heads_first": False, "tree": False},
        # few long conversations without a window, a short chain of drafts
        {"name": "attend long", "op": "attend", "rows": 5, "nodes": 3, "hq": 32, "hkv": 8, "dim": 128, "len": 50001, "page": 64,
         "block": 64, "window": 0, "sinks": 0, "dtype": "bf16", "heads_first": True, "tree": False},
        # wide drafted trees: arithmetic counts as much as memory
        {"name": "attend trees", "op": "attend", "rows": 40, "nodes": 64, "hq": 32, "hkv": 4, "dim": 128, "len": 6000, "page": 32,
         "block": 8, "window": 0, "sinks": 0, "dtype": "bf16", "heads_first": False, "tree": True},
        # chunks of long prompts: bound by arithmetic
        {"name": "attend prompts", "op": "attend", "rows": 3, "nodes": 2000, "hq": 32, "hkv": 8, "dim": 128, "len": 8000,
         "page": 128, "block": 128, "window": 0, "sinks": 0, "dtype": "bf16", "heads_first": False, "tree": False},
        # one token of one conversation over the model's vocabulary: latency
        {"name": "logprobs one", "op": "logprobs", "rows": 1, "vocab": 248320, "given": 1, "top": 20, "dtype": "fp32",
         "temperature": 1.0},
        # a token of every slot, siblings of a tree as the given tokens
        {"name": "logprobs slots", "op": "logprobs", "rows": 352, "vocab": 248320, "given": 4, "top": 5, "dtype": "bf16",
         "temperature": 0.7},
        # drafted tokens of a full server, an odd vocabulary (rows begin anywhere)
        {"name": "logprobs odd", "op": "logprobs", "rows": 2500, "vocab": 50001, "given": 1, "top": 20, "dtype": "fp16",
         "temperature": 1.0},
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "logprobs", "logprobs"])
    if op == "logprobs":
        while True:
            case = {"op": op, "rows": _spread(rng, 1, 2500), "vocab": _spread(rng, 1000, 248320), "given": _spread(rng, 1, 8),
                    "top": rng.choice([0, 1, 5, 20, 64]), "dtype": rng.choice(["fp32", "bf16", "fp16"]),
                    "temperature": rng.choice([1.0, 1.0, 0.7, 1.3])}
            if case["rows"] * case["vocab"] * (2 if case["dtype"] == "fp32" else 1) <= 352 * 248320:
                return case
    dim, dtype, heads_first = rng.choice([64, 128, 256]), rng.choice(["fp16", "bf16"]), rng.random() < 0.5
    page = rng.choice([8, 16, 32, 48, 64, 128])
    block = rng.choice([b for b in (8, 16, 24, 32, 64, 128) if page % b == 0])
    if op == "append":
        while True:
            hq, hkv = rng.choice([(8, 2), (8, 8), (32, 8), (16, 2), (15, 5), (7, 1), (6, 2)])
            case = {"op": op, "rows": _spread(rng, 1, 352), "grow": _spread(rng, 1, 2500), "hq": hq, "hkv": hkv, "dim": dim,
                    "rot": rng.choice([dim, dim // 2, dim // 4]), "len": _spread(rng, 1, 50000), "page": page, "block": block,
                    "pairs": rng.random() < 0.5, "factor": rng.choice([1.0, 1.0, 1.2079, 0.8]), "dtype": dtype,
                    "heads_first": heads_first}
            if case["rows"] * case["grow"] * (hq + hkv) * dim <= 20 * 2500 * 40 * 128:
                return case
    while True:
        hq, hkv = rng.choice([(8, 2), (8, 8), (32, 8), (16, 2), (15, 5), (7, 1), (32, 4)])
        tree = rng.random() < 0.3
        case = {"op": op, "rows": _spread(rng, 1, 352), "nodes": _spread(rng, 1, 200 if tree else 2000), "hq": hq, "hkv": hkv,
                "dim": dim, "len": _spread(rng, 1, 50000), "page": page, "block": block,
                "window": rng.choice([0, 0, 512, _spread(rng, 3, 5000)]), "sinks": rng.choice([0, 1, 4, 16]), "dtype": dtype,
                "heads_first": heads_first, "tree": tree}
        case["len"] = max(case["len"], case["nodes"])
        if not case["window"]:
            case["sinks"] = 0
        # no dearer than the largest listed cases: cache held, scores of the plain form
        keys = case["rows"] * _reach(case)
        if case["rows"] * case["len"] * hkv * dim <= 352 * 8000 * 2 * 256 and keys * hkv * dim <= 5 * 50001 * 8 * 128 \
                and keys * hq * case["nodes"] <= 3 * 8000 * 32 * 2000:
            return case


def _reach(case):
    """The most tokens that a request's newest ones read, themselves among them."""
    return min(case["len"], case["sinks"] + case["window"] + case["nodes"]) if case["window"] else case["len"]


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _shares(n):
    """Numbers in [0, 1), evenly spread: which request has which is the seed's choice, their sum is the case's."""
    return (0.37 + 0.6180339887 * torch.arange(n, dtype=torch.float64, device="cuda")) % 1


def _counts(n, top, g):
    """New tokens a request: half full, the others fewer; in a larger batch one request has none."""
    c = torch.clamp(torch.floor(2 * top * _shares(n)), 1, top).to(torch.int32)
    c[0] = top
    if n > 3:
        c[3] = 0
    return c[torch.randperm(n, generator=g, device="cuda")]


def _lengths(n, top, g):
    """Unequal lengths in [0, top]: most in the upper half, a few short, in a batch the first one full and one empty."""
    u = torch.rand(n, generator=g, device="cuda")
    lens = (top * (0.5 + 0.5 * u)).to(torch.int32)
    lens = torch.where(torch.rand(n, generator=g, device="cuda") < 0.1, (top * u * u).to(torch.int32), lens)
    if n > 1:
        lens[0] = top
    if n > 2:
        lens[n // 2] = 0
    return lens


def _offsets(counts):
    cu = torch.zeros(len(counts) + 1, dtype=torch.int32, device="cuda")
    cu[1:] = torch.cumsum(counts, 0)
    return cu


def _pool(pages, page, hkv, dim, heads_first, g):
    """Codes of a cache [pages, page, hkv, dim], heads or tokens outermost within a page."""
    shape = (pages, hkv, page, dim) if heads_first else (pages, page, hkv, dim)
    pool = torch.empty(shape, dtype=F8, device="cuda")
    flat = pool.view(-1)
    for part in flat.split(1 << 27):
        part.copy_((90 * torch.randn(part.numel(), generator=g, device="cuda")).clamp_(-448, 448))
    return pool.transpose(1, 2) if heads_first else pool


def _trees(counts, cu, g):
    """Parent links (parents first, -1: none) of drafted trees: a few branches at each level."""
    total = int(cu[-1])
    index = torch.arange(total, device="cuda") - torch.repeat_interleave(cu[:-1].long(), counts.long())
    u = torch.rand(total, generator=g, device="cuda")
    parents = torch.floor((index.float() * (0.35 + 0.3 * u))).long()
    return torch.where((index < 2) | (parents >= index), -1, parents)


def _ancestors(parents, cu, words):
    """Ancestor bits [tokens, words] (int32) and depths; each round doubles how far up every token looks."""
    total = parents.shape[0]
    rows = torch.bucketize(torch.arange(total, device="cuda"), cu[1:], right=True)
    base = cu.long()[rows]
    up = torch.where(parents >= 0, base + parents, total)
    up = torch.cat([up, up.new_full((1,), total)])
    bits = torch.zeros(total + 1, words * 32, dtype=torch.bool, device="cuda")
    bits[:total].scatter_(1, (torch.arange(total, device="cuda") - base)[:, None], True)
    for _ in range((words * 32).bit_length()):
        bits = bits | bits[up]
        up = up[up]
    bits = bits[:total]
    packed = (bits.view(total, words, 32) * (1 << torch.arange(32, device="cuda"))).sum(-1)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32), bits.sum(-1) - 1


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    s = {"case": case}
    if op == "logprobs":
        n, vocab = case["rows"], case["vocab"]
        x = torch.empty(n, vocab, dtype=DTYPES[case["dtype"]], device="cuda")
        x.normal_(0, 2.5, generator=g)
        # a few likely tokens, as a language model's rows have; some tokens forbidden by a grammar
        likely = torch.randint(0, vocab, (n, 12), generator=g, device="cuda")
        x.scatter_reduce_(1, likely, (14 + 4 * torch.randn(n, 12, generator=g, device="cuda")).to(x.dtype), "amax")
        x.scatter_(1, torch.randint(0, vocab, (n, 40), generator=g, device="cuda"), float("-inf"))
        given = torch.randint(0, vocab, (n, case["given"]), generator=g, device="cuda")
        given[:, 0] = likely[:, 0]
        if case["given"] > 1:
            given[n // 2, 1:] = -1  # a node with one child
        s.update(x=x, given=given.to(torch.int32), top=case["top"], temperature=case["temperature"])
        return s
    hq, hkv, dim, page, block, dtype = (case[x] for x in ("hq", "hkv", "dim", "page", "block", "dtype"))
    dtype, n = DTYPES[dtype], case["rows"]
    if op == "append":
        counts, start = _counts(n, case["grow"], g), _lengths(n, case["len"], g)
        total = int(counts.sum())
        cu = _offsets(counts)
        row = torch.repeat_interleave(torch.arange(n, device="cuda"), counts.long())
        positions = start[row] + (torch.arange(total, device="cuda") - cu[row])
        first = start // page
        held = (counts + page - 1) // page + 1  # as many as it may touch, wherever it begins
        at = torch.cumsum(held, 0) - held
        pages = int(held.sum()) + 1
        order = torch.randperm(pages, generator=g, device="cuda")
        slots = order[(at[row] + positions // page - first[row]).long()] * page + positions % page
        if total > 2:
            slots[total // 2] = -1  # a token that is not kept
        x = torch.empty(total, (hq + 2 * hkv) * dim, dtype=dtype, device="cuda").normal_(generator=g)  # one projection
        scales = [torch.exp2(torch.randint(-8, -4, (pages, page // block, hkv), generator=g, device="cuda").float())
                  for _ in range(2)]
        s.update(q=x[:, :hq * dim].view(total, hq, dim), k=x[:, hq * dim:(hq + hkv) * dim].view(total, hkv, dim),
                 v=x[:, (hq + hkv) * dim:].view(total, hkv, dim), slots=slots.to(torch.int32),
                 positions=positions.to(torch.int32), factor=case["factor"], pairs=case["pairs"],
                 inv=500000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda").float() / case["rot"]),
                 kc=_pool(pages, page, hkv, dim, case["heads_first"], g), ks=scales[0],
                 vc=_pool(pages, page, hkv, dim, case["heads_first"], g), vs=scales[1])
        return s
    counts = _counts(n, case["nodes"], g)
    cached = _lengths(n, case["len"] - case["nodes"], g)
    lens = cached + counts
    cu = _offsets(counts)
    total = int(cu[-1])
    rows = torch.repeat_interleave(torch.arange(n, device="cuda"), counts.long())
    if case["tree"]:
        mask, depth = _ancestors(_trees(counts, cu, g), cu, (case["nodes"] + 31) // 32)
    else:
        mask, depth = None, torch.arange(total, device="cuda") - cu[rows]
    width = (case["len"] + page - 1) // page
    held = (lens + page - 1) // page
    pages = int(held.sum()) + 2
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    column = torch.arange(width, device="cuda")
    at = (torch.cumsum(held, 0) - held)[:, None] + column
    table = torch.where(column < held[:, None], order[at.clamp(max=pages - 1)], -1).to(torch.int32).contiguous()
    kc, vc = (_pool(pages, page, hkv, dim, case["heads_first"], g) for _ in range(2))
    ks, vs = (torch.exp2(torch.randint(-8, -5, (pages, page // block, hkv), generator=g, device="cuda").float())
              for _ in range(2))
    # memory that no token has filled yet: whatever was there, NaN among it
    nan = torch.tensor(float("nan"), device="cuda").to(F8)
    junk = order[pages - 2:].long()
    part = (lens % page > 0) & (held > 0)
    ends = table.gather(1, (held - 1).clamp(min=0)[:, None].long())[:, 0].clamp(min=0).long()
    tail = part[:, None] & (torch.arange(page, device="cuda") >= (lens % page)[:, None])
    bad_page, bad_at = ends[:, None].expand_as(tail)[tail], torch.arange(page, device="cuda").expand_as(tail)[tail]
    for codes, scales in ((kc, ks), (vc, vs)):
        codes.view(torch.uint8)[junk] = nan.view(torch.uint8)
        codes.view(torch.uint8)[bad_page, bad_at] = nan.view(torch.uint8)
        scales[junk] = float("nan")
    s.update(q=torch.empty(total, hq, dim, dtype=dtype, device="cuda").normal_(generator=g), kc=kc, vc=vc, ks=ks, vs=vs,
             table=table, lens=lens, cu=cu, mask=mask, positions=(cached[rows] + depth).to(torch.int32) if case["tree"] else None,
             scale=dim ** -0.5, window=case["window"], sinks=case["sinks"], nodes=case["nodes"])
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        from hs_guard_b200 import drafts
        if op == "append":
            q = drafts.append_8bit(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["slots"], positions=s["positions"],
                                   inv_freq=s["inv"], interleaved=s["pairs"], rope_scale=s["factor"], q=s["q"])
            return {"q": q, "k": s["kc"], "v": s["vc"], "k_scale": s["ks"], "v_scale": s["vs"]}
        if op == "attend":
            out, lse = drafts.attention_8bit(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["lens"], s["cu"],
                                             s["scale"], max_new=s["nodes"], mask=s["mask"], positions=s["positions"],
                                             window=s["window"], sinks=s["sinks"])
            return {"out": out, "lse": lse}
        r = drafts.token_logprobs(s["x"], s["given"], top=s["top"], temperature=s["temperature"])
        return {"logprobs": r.logprobs, "entropy": r.entropy, "lse": r.lse, "top": r.top, "top_ids": r.top_ids}
    return {"append": _plain_append, "attend": _plain_attend, "logprobs": _plain_logprobs}[op](s)


def _rotated(x, cos, sin, pairs):
    rot = 2 * cos.shape[-1]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs else (x[..., :rot // 2], x[..., rot // 2:rot])
    y, z = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([y, z], -1).flatten(-2) if pairs else torch.cat([y, z], -1)
    return torch.cat([turned, x[..., rot:]], -1), a.abs() + b.abs()


def _scale_of(bound):
    """The smallest power of two, between 2^-100 and 2^120, that brings `bound` to at most 448."""
    m, e = torch.frexp(bound)
    e = torch.where(bound > 0, torch.where(m <= 0.875, e - 9, e - 8), -100)
    return torch.exp2(e.clamp(-100, 120).to(bound.dtype))


def _plain_append(s):
    case = s["case"]
    page, block = case["page"], case["block"]
    angle = s["positions"].double()[:, None] * s["inv"].double()
    cos, sin = ((s["factor"] * f(angle)).float()[:, None] for f in (torch.cos, torch.sin))
    q = _rotated(s["q"].float(), cos, sin, s["pairs"])[0].to(s["q"].dtype)
    kept = s["slots"] >= 0
    slots = s["slots"][kept].long()
    x = s["k"].float()
    rot = 2 * cos.shape[-1]
    k, pair = _rotated(x, cos, sin, s["pairs"])
    reach = torch.cat([pair * torch.tensor(abs(s["factor"]), device="cuda"), x[..., rot:].abs()], -1)
    v = s["v"].float()
    _put(s["kc"], s["ks"], k[kept], reach[kept], slots, page, block)
    _put(s["vc"], s["vs"], v[kept], v[kept].abs(), slots, page, block)
    return {"q": q, "k": s["kc"], "v": s["vc"], "k_scale": s["ks"], "v_scale": s["vs"]}


def _put(codes, scales, x, reach, slots, page, block):
    """Rows x into slots of the cache, in place: scales of the blocks that they reach, rows already there to the new scale."""
    pages, hkv = codes.shape[0], codes.shape[2]
    where = slots // block
    reach = torch.where(torch.isfinite(reach), reach, 0).amax(-1)
    need = torch.zeros(pages * page // block, hkv, device="cuda").index_reduce_(0, where, reach, "amax")
    first = torch.full((pages * page // block,), block, device="cuda").scatter_reduce_(0, where, slots % block, "amin")
    touched = (first < block).nonzero()[:, 0]
    old = scales.view(-1, hkv)[touched]
    fresh = (first[touched] == 0)[:, None]
    new = torch.where(fresh, _scale_of(need[touched]), torch.maximum(old, _scale_of(need[touched])))
    per = page // block
    at_page, at_row = touched // per, (touched % per)[:, None] * block + torch.arange(block, device="cuda")
    rows = codes[at_page[:, None], at_row].float() * (old / new)[:, None, :, None]
    stay = torch.arange(block, device="cuda") < torch.where(fresh[:, 0], 0, first[touched])[:, None]
    codes.view(torch.uint8)[at_page[:, None].expand_as(stay)[stay], at_row[stay]] = rows[stay].to(F8).view(torch.uint8)
    scales.view(-1, hkv)[touched] = new
    y = (x / scales.view(-1, hkv)[where][..., None]).to(F8)
    codes.view(torch.uint8)[slots // page, slots % page] = y.view(torch.uint8)


def _seen(s, kpos, token, node):
    """Which of a request's tokens kpos [rows, keys] its new ones see: [rows, nodes, keys]."""
    lens, cu, window, sinks = s["lens"].long(), s["cu"].long(), s["window"], s["sinks"]
    n = cu[1:] - cu[:-1]
    cached = (lens - n)[:, None]
    drafted = node < n[:, None]
    fresh = kpos - cached  # index among the new tokens
    old, new = (kpos >= 0) & (fresh < 0), (fresh >= 0) & (kpos < lens[:, None])
    if s["mask"] is None:
        qpos = cached + node
        ppos = kpos
        see = old[:, None] | (new[:, None] & (fresh[:, None] <= node[:, None]))
    else:
        qpos = s["positions"].long()[token]
        at = torch.where(new, fresh, 0)
        ppos = torch.where(new, qpos.gather(1, at), kpos)
        word = s["mask"][token].gather(2, (at // 32)[:, None].expand(-1, node.shape[0], -1))
        see = old[:, None] | (new[:, None] & ((word >> (at % 32)[:, None].int()) & 1 != 0))
    if window:
        see = see & ((ppos[:, None] > (qpos - window)[..., None]) | (ppos < sinks)[:, None])
    return see & drafted[..., None], drafted


def _plain_attend(s):
    case = s["case"]
    hq, hkv, dim, nodes, rows, page, block = (case[x] for x in ("hq", "hkv", "dim", "nodes", "rows", "page", "block"))
    lens, cu = s["lens"].long(), s["cu"].long()
    n = cu[1:] - cu[:-1]
    # tokens that a request's new ones can see, padded to the longest
    begin = (lens - n - s["window"] + 1).clamp(min=s["sinks"]) if s["window"] else torch.zeros_like(lens)
    ahead = s["sinks"] if s["window"] else 0
    reach = max(1, _reach(case))
    kpos = begin[:, None] + torch.arange(max(1, reach - ahead), device="cuda")
    kpos = torch.cat([torch.arange(ahead, device="cuda").expand(rows, -1), kpos], 1)
    kpos = torch.where(kpos < lens[:, None], kpos, -1)
    node = torch.arange(nodes, device="cuda")
    token = torch.where(node < n[:, None], cu[:-1, None] + node, 0)
    see, drafted = _seen(s, kpos, token, node)
    there = (kpos >= 0)[..., None, None]
    at = kpos.clamp(min=0)
    page_of = s["table"].long().gather(1, at // page).clamp(min=0)

    def values(codes, scales):
        x = codes[page_of, at % page].float() * scales[page_of, at % page // block][..., None]
        return torch.where(there, x, 0.0).transpose(1, 2)

    q = s["q"][token].float().view(rows, nodes, hkv, hq // hkv, dim).permute(0, 2, 3, 1, 4)
    score = (q.reshape(rows, hkv, -1, dim) @ values(s["kc"], s["ks"]).transpose(-1, -2)) * s["scale"]
    score = score.view(rows, hkv, hq // hkv, nodes, -1).masked_fill_(~see[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(rows, hkv, -1, p.shape[-1]) @ values(s["vc"], s["vs"])).view(rows, hkv, hq // hkv, nodes, dim)
    out = out / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(rows, nodes, hq, dim)
    lse = (top + torch.log(total))[..., 0].permute(0, 3, 1, 2).reshape(rows, nodes, hq)
    return {"out": out[drafted].to(s["q"].dtype), "lse": lse[drafted]}


def _plain_logprobs(s):
    x = s["x"].float() / s["temperature"]
    top = x.amax(-1, keepdim=True)
    z = x - top
    e = torch.exp(z)
    total = e.sum(-1)
    lse = top[:, 0] + torch.log(total)
    entropy = torch.log(total) - torch.where(e > 0, e * z, 0.0).sum(-1) / total
    given = s["given"].long()
    logprobs = torch.where(given >= 0, z.gather(1, given.clamp(min=0)) - torch.log(total)[:, None], 0.0)
    # the type that came in decides between equals: the lowest token first
    best = torch.sort(s["x"].float(), dim=-1, descending=True, stable=True)[1][:, :s["top"]] if s["top"] else given[:, :0]
    return {"logprobs": logprobs, "entropy": entropy, "lse": lse, "top": z.gather(1, best) - torch.log(total)[:, None],
            "top_ids": best.to(torch.int32)}


# ---- 64-bit values --------------------------------------------------------------------------------------------------
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "logprobs":
        x = s["x"].double() / s["temperature"]
        p = torch.softmax(x, -1)
        lse = torch.logsumexp(x, -1)
        given = s["given"].long()
        entropy = -torch.special.xlogy(p, p).sum(-1)
        chosen = torch.where(given >= 0, x.gather(1, given.clamp(min=0)) - lse[:, None], 0.0)
        return {"logprobs": chosen, "entropy": entropy, "lse": lse,
                "top": torch.topk(x, s["top"], -1)[0] - lse[:, None], "top_ids": None}
    if op == "append":
        page, block, hkv = case["page"], case["block"], case["hkv"]
        rot = case["rot"]
        turn = torch.polar(torch.full((), s["factor"], dtype=torch.float64, device="cuda"),
                           s["positions"].double()[:, None, None] * s["inv"].double())

        def rotate(x):
            x = x.double()
            a, b = (x[..., :rot:2], x[..., 1:rot:2]) if s["pairs"] else x[..., :rot].chunk(2, -1)
            z = torch.complex(a.contiguous(), b.contiguous()) * turn
            y = torch.view_as_real(z).flatten(-2) if s["pairs"] else torch.cat([z.real, z.imag], -1)
            # the rule for a block's scale says 32 bits: sums of 16-bit values often lie on a border between two powers
            sizes = (a.abs() + b.abs()).float().mul(torch.tensor(abs(s["factor"]), device="cuda")).double()
            return torch.cat([y, x[..., rot:]], -1), torch.cat([sizes, x[..., rot:].abs()], -1).amax(-1)

        out = {"q": rotate(s["q"])[0]}
        slots = s["slots"].long()
        v = s["v"].double()
        k, k_size = rotate(s["k"])
        for name, codes, scales, y, size in (("k", s["kc"], s["ks"], k, k_size), ("v", s["vc"], s["vs"], v, v.abs().amax(-1))):
            value = codes.double()
            grid = scales.double().clone().view(-1, hkv)
            blocks, inverse = torch.unique(slots[slots >= 0] // block, return_inverse=True)
            size = size[slots >= 0]
            largest = torch.zeros(len(blocks), hkv, dtype=torch.float64, device="cuda")
            largest.scatter_reduce_(0, inverse[:, None].expand_as(size), size, "amax")
            lowest = torch.full((len(blocks),), block, dtype=torch.int64, device="cuda")
            lowest.scatter_reduce_(0, inverse, slots[slots >= 0] % block, "amin")
            need = torch.pow(2.0, torch.ceil(torch.log2(largest / 448)))
            need = torch.where(largest <= 224 * need, need / 2, need)  # a logarithm that came out above a whole number
            old = grid[blocks]
            new = torch.where(lowest[:, None] == 0, need, torch.where(need > old, need, old))
            for i in range(block):  # rows that were there
                moved = ((i < lowest) & (lowest > 0)).nonzero()[:, 0]
                at, row = blocks[moved] * block // page, blocks[moved] * block % page + i
                value[at, row] = value[at, row] * (old / new)[moved][..., None]
            grid[blocks] = new
            kept = slots[slots >= 0]
            value[kept // page, kept % page] = y[slots >= 0] / grid[kept // block][..., None]
            out[name], out[name + "_scale"] = value, grid.view(scales.shape)
        return out
    # request by request over the tokens that it really has
    lens, cu = s["lens"].tolist(), s["cu"].tolist()
    group, page, block, window = case["hq"] // case["hkv"], case["page"], case["block"], s["window"]
    if sum(c * n for n, c in zip(lens, (b - a for a, b in zip(cu, cu[1:])))) * case["hq"] * case["dim"] * 4 > 4e12:
        return None
    outs, lses = [], []
    for b, length in enumerate(lens):
        a, z = cu[b], cu[b + 1]
        if z == a:
            continue
        old = length - (z - a)
        start = min(old, max(0, old - window + 1)) if window else 0
        at = torch.cat([torch.arange(min(start, s["sinks"]), device="cuda"), torch.arange(start, length, device="cuda")])
        where = s["table"][b][at // page].long()
        k, v = (codes[where, at % page].double() * scales[where, at % page // block].double()[..., None]
                for codes, scales in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
        t = torch.arange(z - a, device="cuda")
        qp = old + t if s["mask"] is None else s["positions"][a:z].long()
        if s["mask"] is None:
            new = t <= t[:, None]
        else:
            new = (s["mask"][a:z][:, t // 32] >> (t % 32)) % 2 != 0
        see = torch.cat([torch.ones(z - a, len(at) - (z - a), dtype=torch.bool, device="cuda"), new], 1)
        if window:
            kp = torch.cat([at[:len(at) - (z - a)], qp])
            see = see & ((kp > qp[:, None] - window) | (kp < s["sinks"]))
        for h in range(case["hkv"]):  # a head at a time, for the memory that 64 bits take
            q = s["q"][a:z, h * group:(h + 1) * group].double().transpose(0, 1)
            score = (q @ k[:, h].T * s["scale"]).masked_fill(~see, float("-inf"))
            lse = torch.logsumexp(score, -1)
            weight = torch.exp(score - torch.where(lse == float("-inf"), torch.zeros_like(lse), lse)[..., None])
            outs.append((a, h, (weight @ v[:, h]).transpose(0, 1)))
            lses.append((a, h, lse.T))
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    for whole, parts in ((out, outs), (lse, lses)):
        for a, h, x in parts:
            whole[a:a + len(x), h * group:(h + 1) * group] = x
    return {"out": out, "lse": lse}


# ---- work -----------------------------------------------------------------------------------------------------------
def work(case):
    """Bytes and operations of one pass, from the sizes alone: lengths and counts are 0.7 and 0.75 of their largest on
    average, the shares that prepare() gives them."""
    op, n = case["op"], case["rows"]
    if op == "logprobs":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": n * (case["vocab"] * size + 8 * (case["given"] + case["top"]) + 8), "flops": 5 * n * case["vocab"]}
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    if op == "append":
        t = n * max(1, 0.75 * case["grow"] if n > 1 else case["grow"])
        return {"bytes": t * (4 * hq * dim + 6 * hkv * dim + 8) + 8 * hkv * t / case["block"],
                "flops": t * (6 * hq + 10 * hkv) * dim}
    nodes = max(1, case["nodes"] * (1 if n == 1 else 0.75))
    cached = (case["len"] - case["nodes"]) * (0.75 if n == 1 else 0.7)
    if case["window"]:
        cached = min(cached, case["window"] + case["sinks"])
    pairs = nodes * (cached + nodes / 2 if not case["window"] else min(cached + nodes / 2, case["window"] + case["sinks"]))
    keys = cached + nodes
    return {"bytes": n * (keys * hkv * (2 * dim + 8 / case["block"]) + nodes * hq * (4 * dim + 4)),
            "flops": 4 * n * pairs * hq * dim}
