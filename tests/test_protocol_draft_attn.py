"""A model of the mbarrier protocol of draft_attn_kernel (hs-guard_b200/csrc/draft_attn.cuh, attention of drafted trees),
checked on the CPU under random interleavings of its roles.

Roles, in the kernel's order of waits and arrivals (tile g of the piece uses S buffer g % NS):
  * K warp: per item Q into its ring (`q_empty` -> `q_full`), per tile K (`k_empty` -> `k_full`);
  * V warp: per item its description (`item_empty` -> `item_full`, two slots), per tile V (`v_empty` -> `v_full`);
  * S warp: waits `k_full`, at an item's first tile `q_full`, and `pv_done` of tile g - NS; S_g completes later and then
    arrives on `s_full`, `k_empty` and, after an item's last tile, `q_empty`;
  * P V warp: waits `v_full`, arrives on `v_there`, at an item's first tile waits for the last one's `o_free`, waits
    `p_full`; P V_g completes later and then arrives on `pv_done` and `v_empty`;
  * softmax warps, two groups (even and odd tiles) of WARPS warps: wait `item_full`; per tile of theirs `s_full`, the other
    group's `m_full` of tile g - 1, on a raised maximum `pv_done` of tile g - 1, for a tile whose V is mended `v_there`;
    arrive on their `m_full` and, with P written over S, on `p_full`. The group without the item's last tile arrives on
    `ml_full`; the other waits for that and for `pv_done` of the last tile, reads O and arrives on `o_free`. Both arrive on
    `item_empty`.
A wait tells a phase by its parity, so it must find the phase running or just completed: the model reports a barrier that is
a phase behind (the wait would return at once) or two ahead (it would never return). Every access checks what it finds.
"""
import random

import pytest

WARPS = 2  # of a group: the kernel's four drift apart no differently


class Bar:
    def __init__(self, name, count):
        self.name, self.count, self.arrivals, self.completed = name, count, 0, 0

    def arrive(self):
        self.arrivals += 1
        if self.arrivals == self.count:
            self.arrivals, self.completed = 0, self.completed + 1


class Aliased(Exception):
    pass


def wait(bar, phase):
    while True:
        if bar.completed < phase or bar.completed > phase + 1:
            raise Aliased(f"{bar.name}: waiting for phase {phase} after {bar.completed} completed")
        if bar.completed == phase + 1:
            return
        yield


def run(seed, broken=None):
    rng = random.Random(seed)
    NS, kb, vb, qb = rng.choice([3, 4]), rng.choice([2, 3, 6]), rng.choice([2, 3, 6]), rng.choice([1, 2])
    sizes = [rng.choice([1, 1, 2, 3, 5, 9]) for _ in range(rng.randint(1, 8))]
    item_of = [k for k, n in enumerate(sizes) for _ in range(n)]
    first = [sum(sizes[:k]) for k in range(len(sizes))]
    n = len(item_of)
    special = [rng.random() < 0.4 for _ in range(n)]
    begins = [g == first[item_of[g]] for g in range(n)]
    ends = [g == first[item_of[g]] + sizes[item_of[g]] - 1 for g in range(n)]

    def bars(name, size, count=1):
        return [Bar(f"{name}[{i}]", count) for i in range(size)]

    k_full, k_empty, v_full, v_empty = (bars(x, s) for x, s in (("k_full", kb), ("k_empty", kb), ("v_full", vb), ("v_empty", vb)))
    q_full, q_empty = bars("q_full", qb), bars("q_empty", qb)
    s_full, p_full, pv_done, v_there = bars("s_full", NS), bars("p_full", NS, WARPS), bars("pv_done", NS), bars("v_there", NS)
    m_full = [[Bar(f"m_full[{x}][{w}]", 1) for w in range(WARPS)] for x in range(2)]
    item_full, item_empty, ml_full = bars("item_full", 2), bars("item_empty", 2, 2 * WARPS), bars("ml_full", 2, WARPS)
    o_free = Bar("o_free", WARPS)
    K, V, Q, items = [None] * kb, [None] * vb, [None] * qb, [None, None]
    S = [[None] * WARPS for _ in range(NS)]  # ("S" or "P", tile) of a warp's lanes
    M = [[None] * WARPS for _ in range(2)]
    ML = [[None] * WARPS for _ in range(2)]
    mended, O, reading = [0] * n, [], set()
    later = {"copy": [], "s": [], "pv": []}  # copies land in any order, each warp's products in the order of issue
    state = {"O": O, "done": 0}

    def land(where, at, what, bar):
        def f():
            where[at] = what
            bar.arrive()
        later["copy"].append(f)

    def k_warp():
        for g in range(n):
            if begins[g]:
                k = item_of[g]
                if k >= qb:
                    yield from wait(q_empty[k % qb], k // qb - 1)
                land(Q, k % qb, k, q_full[k % qb])
            if g >= kb:
                yield from wait(k_empty[g % kb], g // kb - 1)
            land(K, g % kb, g, k_full[g % kb])
            yield

    def v_warp():
        for g in range(n):
            if begins[g]:
                k = item_of[g]
                if k >= 2 and broken != "item":
                    yield from wait(item_empty[k & 1], k // 2 - 1)
                items[k & 1] = k
                item_full[k & 1].arrive()
            if g >= vb:
                yield from wait(v_empty[g % vb], g // vb - 1)
            land(V, g % vb, g, v_full[g % vb])
            yield

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
            v_there[g % NS].arrive()
            if begins[g] and k > 0 and broken != "o_free":
                yield from wait(o_free, k - 1)
            yield from wait(p_full[g % NS], g // NS)

            def done(g=g, k=k):
                assert V[g % vb] == g and S[g % NS] == [("P", g)] * WARPS, "P V on another tile's operands"
                assert mended[g] == (WARPS if special[g] else 0), "P V before V was mended"
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
                yield from wait(s_full[g % NS], g // NS)
                assert S[g % NS][w] == ("S", g)
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
                assert S[g % NS][w] == ("S", g)
                S[g % NS][w] = ("P", g)
                if special[g]:
                    if broken == "v_there":
                        yield from wait(v_full[g % vb], g // vb)
                    else:
                        yield from wait(v_there[g % NS], g // NS)
                    assert V[g % vb] == g, "another tile's V mended"
                    mended[g] += 1
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
            reading.add((x, w))
            yield
            assert state["O"] == list(range(first[k], last + 1)) and items[k & 1] == k
            reading.discard((x, w))
            o_free.arrive()
            item_empty[k & 1].arrive()

    roles = [k_warp(), v_warp(), s_warp(), pv_warp()] + [softmax(x, w) for x in range(2) for w in range(WARPS)]
    weight = [rng.choice([1, 1, 5, 20]) for _ in roles] + [rng.choice([1, 5]) for _ in range(3)]
    idle = 0
    while roles or any(later.values()):
        choices = list(range(len(roles))) + [("copy", "s", "pv")[i] for i in range(3) if later[("copy", "s", "pv")[i]]]
        pick = rng.choices(choices, [weight[c] if isinstance(c, int) else weight[-1] for c in choices])[0]
        idle += 1
        assert idle < 200000, "no progress"
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


@pytest.mark.parametrize("broken", ["item", "s", "o_free", "v_there"])
def test_the_model_catches(broken):
    """A description overwritten early, S issued without waiting for P V, O not waited for, V waited for by its ring."""
    caught = 0
    for seed in range(200):
        try:
            run(seed, broken)
        except (AssertionError, Aliased):
            caught += 1
    assert caught
