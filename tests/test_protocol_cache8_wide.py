"""A model of the mbarrier protocol of attn8_wide_kernel (hs-guard_b200/csrc/cache8_wide.cuh, attention of many rows over a cache in
8 bits), checked on the CPU under random interleavings of its roles.

Roles, in the kernel's order of waits and arrivals (tile g of the piece uses S buffer g % NS and place g % 8 of scales and of V's
reports):
  * K warp: per tile K (`k_empty` -> `k_full`) and its scales (`sc_full`, no wait of their own);
  * V warp: per item its description and the queries (`item_empty`, `q_empty` -> `q_full`, `item_full`), per tile V's codes into the
    staging ring (`st_empty` -> `st_full`);
  * converting warps: wait `st_full` and `v_empty`, report a NaN (four places of items), arrive on `st_empty`, `v_full`, `v_seen`;
  * S warp: waits `k_full`, at an item's first tile `q_full`, and `pv_done` of tile g - NS; S_g completes later and then
    arrives on `s_full`, `k_empty` and, after an item's last tile, `q_empty`;
  * P V warp: waits `v_full`, at an item's first tile for the last one's `o_free`, `p_full`; P V_g completes later and then
    arrives on `pv_done` and `v_empty`;
  * softmax warps, two groups (even and odd tiles): wait `item_full`; per tile of theirs `sc_full`, `s_full`, the other group's `m_full`
    of tile g - 1, on a raised maximum `pv_done` of tile g - 1, for a tile that not every row sees alike `v_seen`; arrive on their
    `m_full` and, with P written over S, on `p_full`. The group without the item's last tile arrives on `ml_full`; the other waits
    for that and for `pv_done` of the last tile, reads the report and O and arrives on `o_free`. Both arrive on `item_empty`.
A wait tells a phase by its parity, so it must find the phase running or just completed: the model reports a barrier that is
a phase behind (the wait would return at once) or two ahead (it would never return). Every access checks what it finds.
"""
import os
import random
import re

import pytest

from test_protocol_draft_attn import Aliased, Bar, wait

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hs-guard_b200", "csrc", "cache8_wide.cuh")
WARPS = 2  # of a group, and of those that convert: the kernel's four drift apart no differently
PLACES, K_BUFS, STAGED = 8, 3, 2
VARIANTS = [(64, 2), (64, 3), (128, 2), (128, 3), (256, 2), (256, 3)]  # head dim, e4m3 numbers of a query's element


def rings(dim, parts):
    """S buffers, Q and V buffers."""
    return (4 if dim == 256 else 3), (2 if dim == 64 or (dim == 128 and parts == 2) else 1), (1 if dim == 256 and parts == 3 else 2)


def test_the_models_sizes_are_the_kernels():
    text = open(SOURCE).read()
    assert "constexpr int W8_PLACES = %d;" % PLACES in text
    assert "constexpr int W8_K_BUFS = %d, W8_STAGED = %d;" % (K_BUFS, STAGED) in text
    body = {n: re.search(r"w8_%s\(int dim[^)]*\) \{ return (.*?); \}" % n, text).group(1) for n in ("scores", "q_bufs", "v_bufs")}
    assert body == {"scores": "dim == 256 ? 4 : 3", "q_bufs": "dim == 64 || (dim == 128 && parts == 2) ? 2 : 1",
                    "v_bufs": "dim == 256 && parts == 3 ? 1 : 2"}


def run(seed, broken=None):
    rng = random.Random(seed)
    (NS, qb, vb), kb, sb, places = rings(*rng.choice(VARIANTS)), K_BUFS, STAGED, PLACES
    reports = 4
    if broken == "places":
        places = 4
    if broken == "reports":
        reports = 1
    sizes = [rng.choice([1, 1, 1, 2, 3, 5, 9, 20]) for _ in range(rng.randint(1, 10))]
    item_of = [k for k, n in enumerate(sizes) for _ in range(n)]
    first = [sum(sizes[:k]) for k in range(len(sizes))]
    n = len(item_of)
    special = [rng.random() < 0.4 for _ in range(n)]
    nan = [special[g] and rng.random() < 0.5 for g in range(n)]
    begins = [g == first[item_of[g]] for g in range(n)]
    ends = [g == first[item_of[g]] + sizes[item_of[g]] - 1 for g in range(n)]

    def bars(name, size, count=1):
        return [Bar(f"{name}[{i}]", count) for i in range(size)]

    k_full, k_empty, st_full, st_empty = bars("k_full", kb), bars("k_empty", kb), bars("st_full", sb), bars("st_empty", sb, WARPS)
    v_full, v_empty, q_full, q_empty = bars("v_full", vb, WARPS), bars("v_empty", vb), bars("q_full", qb), bars("q_empty", qb)
    s_full, p_full, pv_done = bars("s_full", NS), bars("p_full", NS, WARPS), bars("pv_done", NS)
    sc_full, v_seen = bars("sc_full", places), bars("v_seen", places, WARPS)
    m_full = [[Bar(f"m_full[{x}][{w}]", 1) for w in range(WARPS)] for x in range(2)]
    item_full, item_empty, ml_full = bars("item_full", 2), bars("item_empty", 2, 2 * WARPS), bars("ml_full", 2, WARPS)
    o_free = Bar("o_free", WARPS)
    K, Q, items, scales = [None] * kb, [None] * qb, [None, None], [None] * places
    staged, V = [None] * sb, [[None] * WARPS for _ in range(vb)]
    S = [[None] * WARPS for _ in range(NS)]  # ("S" or "P", tile) of a warp's lanes
    M = [[None] * WARPS for _ in range(2)]
    ML = [[None] * WARPS for _ in range(2)]
    report = [-1] * reports
    reading = set()
    later = {"copy": [], "s": [], "pv": []}  # copies land in any order, each warp's products in the order of issue
    state = {"O": [], "done": 0}

    def land(where, at, what, bar):
        def f():
            where[at] = what
            bar.arrive()
        later["copy"].append(f)

    def k_warp():
        for g in range(n):
            if g >= kb:
                yield from wait(k_empty[g % kb], g // kb - 1)
            land(K, g % kb, g, k_full[g % kb])
            yield
            scales[g % places] = g
            sc_full[g % places].arrive()
            yield

    def v_warp():
        for g in range(n):
            if begins[g]:
                k = item_of[g]
                if k >= 2 and broken != "item":
                    yield from wait(item_empty[k & 1], k // 2 - 1)
                if k >= qb:
                    yield from wait(q_empty[k % qb], k // qb - 1)
                items[k & 1] = k
                land(Q, k % qb, k, q_full[k % qb])
                item_full[k & 1].arrive()
            if g >= sb:
                yield from wait(st_empty[g % sb], g // sb - 1)
            land(staged, g % sb, g, st_full[g % sb])
            yield

    def convert(w):
        for g in range(n):
            yield from wait(st_full[g % sb], g // sb)
            if g >= vb:
                yield from wait(v_empty[g % vb], g // vb - 1)
            assert staged[g % sb] == g, "another tile's codes"
            V[g % vb][w] = g
            if nan[g] and w == g % WARPS:
                report[item_of[g] % reports] = item_of[g]
            yield
            assert staged[g % sb] == g, "codes overwritten while they are read"
            st_empty[g % sb].arrive()
            v_full[g % vb].arrive()
            v_seen[g % places].arrive()

    def s_warp():
        for g in range(n):
            k = item_of[g]
            yield from wait(k_full[g % kb], g // kb)
            if begins[g]:
                yield from wait(q_full[k % qb], k // qb)
            if g >= NS and broken != "s":
                yield from wait(pv_done[g % NS], g // NS - 1)

            def done(g=g, k=k):
                assert K[g % kb] == g and Q[k % qb] == k, "S on another tile's operands"
                assert all(x is None or x == ("P", g - NS) for x in S[g % NS]) and state["done"] > g - NS, "S over a live buffer"
                S[g % NS] = [("S", g)] * WARPS
                s_full[g % NS].arrive()
                k_empty[g % kb].arrive()
                if ends[g]:
                    q_empty[k % qb].arrive()
            later["s"].append(done)
            yield

    def pv_warp():
        for g in range(n):
            k = item_of[g]
            yield from wait(v_full[g % vb], g // vb)
            if begins[g] and k > 0 and broken != "o_free":
                yield from wait(o_free, k - 1)
            yield from wait(p_full[g % NS], g // NS)

            def done(g=g):
                assert V[g % vb] == [g] * WARPS and S[g % NS] == [("P", g)] * WARPS, "P V on another tile's operands"
                assert not (begins[g] and reading), "O overwritten while it is read"
                state["O"] = [g] if begins[g] else state["O"] + [g]
                state["done"] = g + 1
                pv_done[g % NS].arrive()
                v_empty[g % vb].arrive()
            later["pv"].append(done)
            yield

    def softmax(x, w):
        for k, size in enumerate(sizes):
            yield from wait(item_full[k & 1], k // 2)
            for g in range(first[k], first[k] + size):
                assert items[k & 1] == k, "another item's description"
                if g & 1 != x:
                    continue
                yield from wait(sc_full[g % places], g // places)
                yield from wait(s_full[g % NS], g // NS)
                assert S[g % NS][w] == ("S", g) and scales[g % places] == g, "another tile's scores or scales"
                yield
                if g > 0:
                    yield from wait(m_full[x ^ 1][w], (g - 1) // 2)
                    assert M[x ^ 1][w] == g - 1
                M[x][w] = g
                m_full[x][w].arrive()
                if not begins[g] and rng.random() < 0.3:  # the maximum rises: O is rescaled
                    yield from wait(pv_done[(g - 1) % NS], (g - 1) // NS)
                    assert state["O"] == list(range(first[k], g))
                yield
                assert S[g % NS][w] == ("S", g) and scales[g % places] == g, "scales overwritten while they are read"
                S[g % NS][w] = ("P", g)
                if special[g]:
                    yield from wait(v_seen[g % places], g // places)
                    assert V[g % vb] == [g] * WARPS
                p_full[g % NS].arrive()
            last = first[k] + size - 1
            if last & 1 != x:
                ML[k & 1][w] = k
                ml_full[k & 1].arrive()
                item_empty[k & 1].arrive()
                continue
            yield from wait(ml_full[k & 1], k // 2)
            assert ML[k & 1][w] == k
            yield from wait(pv_done[last % NS], last // NS)
            yield
            assert (report[k % reports] == k) == any(nan[first[k]:last + 1]), "a report lost"
            reading.add((x, w))
            yield
            assert state["O"] == list(range(first[k], last + 1)) and items[k & 1] == k
            reading.discard((x, w))
            o_free.arrive()
            yield
            assert items[k & 1] == k, "a description overwritten while rows are mended"
            item_empty[k & 1].arrive()

    roles = [k_warp(), v_warp(), s_warp(), pv_warp()] + [convert(w) for w in range(WARPS)] + \
            [softmax(x, w) for x in range(2) for w in range(WARPS)]
    weight = [rng.choice([1, 1, 5, 20]) for _ in roles] + [rng.choice([1, 5])]
    idle = 0
    while roles or any(later.values()):
        choices = list(range(len(roles))) + [x for x in later if later[x]]
        pick = rng.choices(choices, [weight[c] if isinstance(c, int) else weight[-1] for c in choices])[0]
        idle += 1
        assert idle < 400000, "no progress"
        if pick == "copy":
            later["copy"].pop(rng.randrange(len(later["copy"])))()
        elif isinstance(pick, str):
            later[pick].pop(0)()
        else:
            try:
                next(roles[pick])
            except StopIteration:
                roles.pop(pick)
                weight.pop(pick)
    assert state["done"] == n


@pytest.mark.parametrize("block", range(20))
def test_random_interleavings(block):
    for seed in range(block * 25, block * 25 + 25):
        run(seed)


@pytest.mark.parametrize("broken", ["item", "s", "o_free", "places", "reports"])
def test_the_model_catches(broken):
    """A description overwritten early, S issued without waiting for P V, O not waited for, too few places of scales or reports."""
    caught = 0
    for seed in range(300):
        try:
            run(seed, broken)
        except (AssertionError, Aliased):
            caught += 1
    assert caught
