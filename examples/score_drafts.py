"""Draft scoring on one softmax layer of the classifier: trees of drafted tokens attended before any is accepted.

    python examples/score_drafts.py

Part 1: over the rings of live conversations. A guard engine has read conversations of unequal lengths; a host model
drafts a tree for each, and the layer attends all of them over the conversations' own 512-token rings, which stay as they
are. Part 2: over a paged cache without a window. Prompts go into pages, then each tick attends drafted trees, accepts one
branch of each and stores its keys and values. The layer's norm weights, rotation and head layout are the model's (random
initialisation); its inputs are random rows of the fused projection (q | gate per head, k, v). Every result is compared
with a 64-bit computation, and the paths are timed.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from hs_guard_b200 import DEFAULT, drafts, weights  # noqa: E402
from hs_guard_b200.engine import SlotEngine  # noqa: E402


class Layer:
    """What one softmax layer does to projected rows: norms and rotation, and the split of the fused projection."""

    def __init__(self, lay, inv_freq, cfg=DEFAULT):
        self.q_norm, self.k_norm, self.inv_freq, self.cfg = lay["q_norm"], lay["k_norm"], inv_freq, cfg
        self.scale = cfg.attn_head_dim ** -0.5

    def split(self, proj):
        c = self.cfg
        gated, kv = 2 * c.attn_heads * c.attn_head_dim, c.kv_heads * c.attn_head_dim
        return (proj[:, :gated].unflatten(1, (c.attn_heads, 2 * c.attn_head_dim))[..., :c.attn_head_dim],
                proj[:, gated:gated + kv].unflatten(1, (c.kv_heads, c.attn_head_dim)),
                proj[:, gated + kv:].unflatten(1, (c.kv_heads, c.attn_head_dim)))

    def rows(self, proj, positions):
        """Rotated q and k, and v, of projected rows, fp16."""
        return drafts.norm_rope(*self.split(proj), self.q_norm, self.k_norm, self.inv_freq, positions, self.cfg.rms_eps,
                                torch.float16)

    def store(self, proj, positions, k_cache, v_cache, slots):
        """The same for committed tokens, keys and values going straight into the pages; returns q."""
        return drafts.norm_rope_store(*self.split(proj), self.q_norm, self.k_norm, self.inv_freq, positions,
                                      self.cfg.rms_eps, k_cache, v_cache, slots)


def draft_trees(sizes, seed):
    """Parent links of drafted trees (a child of one of the three latest tokens, or of the conversation) and offsets."""
    g = torch.Generator().manual_seed(seed)
    parents = [max(-1, i - 1 - int(torch.randint(0, 3, (1,), generator=g))) for n in sizes for i in range(n)]
    cu = torch.tensor([0] + list(torch.cumsum(torch.tensor(sizes), 0)), dtype=torch.int32)
    return torch.tensor(parents, dtype=torch.int32).cuda(), cu.cuda()


def branch(parents, cu, request, node):
    """A drafted token's branch, oldest first, as indexes within its request."""
    path, first = [], int(cu[request])
    while node >= 0:
        path.append(node)
        node = int(parents[first + node])
    return path[::-1]


def reference(q, k, v, old_k, old_v, old_pos, parents, cu, positions, request, scale, window):
    """One request's attention in 64 bits: every drafted token over its visible cached keys and its own branch."""
    first, outs = int(cu[request]), []
    for t in range(first, int(cu[request + 1])):
        low = int(positions[t]) - window if window else -1
        keep = old_pos > low
        nodes = [first + j for j in branch(parents, cu, request, t - first) if int(positions[first + j]) > low]
        keys = torch.cat([old_k[keep], k[nodes]]).double()
        values = torch.cat([old_v[keep], v[nodes]]).double()
        heads = q[t].double().unflatten(0, (keys.shape[1], -1))
        p = torch.softmax(torch.einsum("hgd,nhd->hgn", heads, keys) * scale, -1)
        outs.append(torch.einsum("hgn,nhd->hgd", p, values).flatten(0, 1))
    return torch.stack(outs)


def timed(f, times=20):
    f()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    for _ in range(times):
        f()
    end.record()
    end.synchronize()
    return begin.elapsed_time(end) / times * 1e3


def over_rings(engine, layer, slots, sizes, seed=0, layer_index=0, check=True):
    """Part 1 for a live engine; returns (largest error against 64 bits, microseconds a tick)."""
    cfg = engine.cfg
    k_cache, v_cache, table, lens = drafts.ring_cache(engine, layer_index, slots)
    parents, cu = draft_trees(sizes, seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    proj = torch.randn(int(cu[-1]), cfg.attn_in_rows, generator=g, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def tick():
        positions, mask = drafts.plan_tree(parents, cu, lens, max(sizes), err)
        q, k, v = layer.rows(proj, positions)
        out, lse = drafts.tree_attention(q, k, v, k_cache, v_cache, table, lens, cu, layer.scale, max(sizes), mask,
                                         positions, cfg.window, err=err)
        return positions, q, k, v, out

    positions, q, k, v, out = tick()
    drafts.raise_device_error(err)
    worst = 0.0
    if check:
        pools = engine.pools()
        for b, slot in enumerate(slots):
            n = int(engine.length[slot])
            pos = torch.arange(max(0, n - cfg.window), n, device="cuda")
            old_k, old_v = (pools[x][layer_index, slot][:, pos % cfg.window].transpose(0, 1) for x in ("ring_k", "ring_v"))
            ref = reference(q, k, v, old_k, old_v, pos, parents, cu, positions, b, layer.scale, cfg.window)
            worst = max(worst, float((out[int(cu[b]):int(cu[b + 1])].double() - ref).abs().max()))
    us = timed(tick)
    drafts.ring_done(engine)  # the engine's next tick writes these rings
    return worst, us


def over_pages(layer, prompts, sizes, ticks, page_size=16, seed=0):
    """Part 2: returns (largest error against 64 bits, lengths at the end)."""
    cfg = layer.cfg
    rows, room = len(prompts), max(prompts) + ticks * max(sizes)
    cache = drafts.DraftCache(1, rows, rows * (-(-room // page_size)), page_size, room, cfg.kv_heads, cfg.attn_head_dim)
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = cache.advance(torch.tensor(prompts, dtype=torch.int32).cuda(), sum(prompts))
    proj = torch.randn(sum(prompts), cfg.attn_in_rows, generator=g, device="cuda")
    layer.store(proj, t.positions, cache.k[0], cache.v[0], t.slots)
    worst = 0.0
    for tick in range(ticks):
        parents, cu = draft_trees(sizes, seed + tick)
        positions, mask = drafts.plan_tree(parents, cu, cache.lens, max(sizes), cache.err)
        proj = torch.randn(sum(sizes), cfg.attn_in_rows, generator=g, device="cuda")
        q, k, v = layer.rows(proj, positions)
        out, lse = cache.attend(0, q, k, v, cu, layer.scale, max(sizes), mask, positions)
        for b, n in enumerate(cache.lens.tolist()):
            pos = torch.arange(n, device="cuda")
            at = cache.table[b][pos // page_size].long(), pos % page_size
            ref = reference(q, k, v, cache.k[0][at], cache.v[0][at], pos, parents, cu, positions, b, layer.scale, 0)
            worst = max(worst, float((out[int(cu[b]):int(cu[b + 1])].double() - ref).abs().max()))
        # accept the branch that ends in the token whose first head looks most at few keys (any rule does here)
        paths = [branch(parents, cu, b, int(lse[int(cu[b]):int(cu[b + 1]), 0].argmax())) for b in range(rows)]
        accepted = torch.tensor([len(p) for p in paths], dtype=torch.int32).cuda()
        t = cache.advance(accepted, int(accepted.sum()))
        source = torch.tensor([int(cu[b]) + i for b, p in enumerate(paths) for i in p], dtype=torch.int32).cuda()
        cache.store(0, k, v, t.slots, source)
    cache.raise_device_error()
    return worst, cache.lens.tolist()


def main():
    engine = SlotEngine(weights.random_state_dict(0), 4)
    g = torch.Generator().manual_seed(1)
    contexts = [700, 41, 513, 64]
    engine.step([(s, torch.randint(0, 1000, (n,), generator=g).tolist()) for s, n in enumerate(contexts)])
    index = DEFAULT.layer_types.index("full_attention")
    layer = Layer(engine.weights["layers"][index], engine.weights["inv_freq"])
    worst, us = over_rings(engine, layer, [2, 0, 3], [12, 7, 15])
    print(f"rings: trees of 12, 7 and 15 tokens over 513, 700 and 64 cached ones, worst error {worst:.1e}, {us:.0f} us a tick")
    worst, lens = over_pages(layer, [300, 17, 1200], [9, 5, 16], 3)
    print(f"pages: three ticks over prompts of 300, 17 and 1200 tokens, worst error {worst:.1e}, lengths now {lens}")
    engine.close()


if __name__ == "__main__":
    main()
