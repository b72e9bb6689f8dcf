"""Draft scoring on a B200 where it can go wrong: weights far below the largest one, tokens of no request, rings without
room, page ids outside their range, caches used on several streams, gradients, and the widest shapes.

Tolerances are those of test_gpu_drafts.py unless a test says otherwise; all were derived before the first run."""
import math

import numpy as np
import pytest
import torch

from test_gpu_drafts import BF16, D, F16, F32, TINY, U, Case, dev, err_word  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- attention: many small weights beside a large one ---------------------------------------------------------------
@pytest.mark.parametrize("dim,dtype,nats,requests,keys", [
    (64, F16, 10.0, 1, 40000), (64, F16, 17.0, 1, 40000), (128, F16, 14.0, 1, 60000), (256, F16, 17.0, 1, 30000),
    (64, F16, 12.0, 296, 19840), (128, F16, 17.0, 296, 19840), (256, F16, 14.0, 296, 9920), (128, BF16, 17.0, 296, 19840),
    (128, F16, 17.0, 296, 2944)])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
def test_tree_attention_many_small_weights_beside_a_large_one(D, dim, dtype, nats, requests, keys, where):
    """One key with V = 0 and `nats` more than all others, which have V = c: the output is n e^-nats / (1 + n e^-nats) c, made
    of the small weights alone. They are at least 2^-25 of the largest (17.3 nats), which fp16 still holds to 2^-11 beside it.
    296 requests on the same pages: items of an even number of pieces, so that none is cut; one request: all are cut.

    Tolerance: that of any attention, and 2^-23 a step of 16 keys for the accumulation of equal terms in fp32, relative."""
    hq, hkv, page = 8, 8 if requests == 1 else 1, 64
    g = torch.Generator(device="cuda").manual_seed(dim)
    pages = -(-keys // page)
    c = torch.randn(hkv, dim, generator=g, device="cuda").to(dtype)
    kc = torch.zeros(pages, page, hkv, dim, device="cuda", dtype=dtype)
    vc = c.expand(pages, page, hkv, dim).contiguous()
    at = {"first": 0, "middle": keys // 2, "last": keys - 1}[where]
    kc[at // page, at % page, :, 0] = nats
    vc[at // page, at % page] = 0
    q = torch.zeros(requests, hq, dim, device="cuda", dtype=dtype)
    q[:, :, 0] = 8.0  # scale 1/8: scores are `nats` and 0
    k, v = torch.zeros(requests, hkv, dim, device="cuda", dtype=dtype), c.expand(requests, hkv, dim).contiguous()
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(requests, pages).contiguous()
    err = err_word()
    out, lse = D.tree_attention(q, k, v, kc, vc, table, dev([keys] * requests), dev(range(requests + 1)), 0.125, 1, err=err)
    assert int(err.item()) == 0
    small = keys * math.exp(-nats)  # all cached keys but one, and the drafted token itself
    share = small / (1 + small)
    ref = (share * c.double()).repeat_interleave(hq // hkv, 0)
    u, ds, steps = U[dtype], dim * 2.0 ** -24 * nats, keys / 16 * 2.0 ** -23
    tol = (u + u + 2 * ds + steps) * ref.abs() + TINY[dtype]
    worst = float(((out.double() - ref).abs() / tol).max())
    assert worst <= 1, f"{worst:.1f} times the tolerance"
    want = nats + math.log1p(small)
    assert float((lse.double() - want).abs().max()) <= ds + 4e-6 * (1 + want) + steps


# ---- advance_tables: rings without room, counters out of range ------------------------------------------------------
@pytest.mark.parametrize("lens,delta,ring,counters,new,new_counters,new_ring,code", [
    # four free entries of four: nothing can come back, the append takes two
    ([32, 0], [-32, 32], [5, 6, 7, 8], [8, 12], [32, 32], [10, 12], [5, 6, 7, 8], 5),
    # two places: the first return fits, the second does not, the third is behind it
    ([32, 32, 16], [-32, -17, -16], [5, 6, -1, -1], [4, 6], [0, 32, 16], [4, 8], [5, 6, 0, 1], 5),
    # exactly full afterwards
    ([32, 32], [-32, 0], [5, 6, -1, -1], [4, 6], [0, 32], [4, 8], [5, 6, 0, 1], 0),
    # taking back within a page needs no place
    ([32, 30], [-3, -13], [5, 6], [6, 8], [29, 17], [6, 8], [5, 6], 0),
    # returns behind an append that is not served, in a ring that goes round
    ([20, 40], [100, -40], [5, -1, -1, -1, 6], [4, 6], [20, 0], [4, 9], [5, 2, 3, 4, 6], 0),
    # counters that cannot be: no page moves, what needs none is served
    ([32, 0, 20, 3], [-32, 32, 5, -3], [5, 6, 7, 8], [-1, 3], [32, 0, 25, 3], [-1, 3], [5, 6, 7, 8], 5),
    ([32, 0, 20, 3], [-32, 32, 5, -3], [5, 6, 7, 8], [3, 2], [32, 0, 25, 3], [3, 2], [5, 6, 7, 8], 5),
    ([32, 0, 20, 3], [-32, 32, 5, -3], [5, 6, 7, 8], [0, 5], [32, 0, 25, 3], [0, 5], [5, 6, 7, 8], 5)])
def test_advance_tables_ring_without_room(D, lens, delta, ring, counters, new, new_counters, new_ring, code):
    page, width = 16, 12
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for b, n in enumerate(lens):
        held = -(-n // page)
        table[b, :held] = torch.arange(at, at + held, dtype=torch.int32)
        at += held
    want, taken, listed = table.clone(), 0, []
    for b, n in enumerate(new):
        for p in range(-(-lens[b] // page), -(-n // page)):
            want[b, p] = ring[(counters[0] + taken) % len(ring)]
            taken += 1
        listed += [(int(want[b, p // page]) * page + p % page, b, p) for p in range(lens[b], n)]
    d_table, d_ring = table.cuda(), dev(ring)
    for _ in range(2):  # the same call again gives the same result
        err = err_word()
        t = D.advance_tables(dev(lens), dev(delta), d_table, d_ring, dev(counters, torch.int64), page, 64, err)
        assert int(err.item()) == code
        assert t.lens.tolist() == new and t.counters.tolist() == new_counters
        assert d_ring.tolist() == new_ring and torch.equal(d_table.cpu(), want)
        none = [(-1, -1, -1)] * (64 - len(listed))
        assert list(zip(t.slots.tolist(), t.rows.tolist(), t.positions.tolist())) == listed + none


@pytest.mark.parametrize("rows,places", [(4000, 9000), (4000, 0), (3000, 1), (700, 10 ** 6)])
def test_advance_tables_many_returns_into_few_places(D, rows, places):
    """Several requests a thread and several thread blocks: served up to the first return without a place."""
    page = 8
    g = torch.Generator().manual_seed(rows)
    lens = torch.randint(0, 60, (rows,), generator=g).tolist()
    delta = torch.randint(-60, 20, (rows,), generator=g).tolist()
    held = [-(-n // page) for n in lens]
    width, used = 12, sum(held)
    free = used // 3
    size = free + min(places, used)
    head = 7 * size + size // 2
    order = torch.randperm(used + free, generator=g).tolist()
    table, at = torch.full((rows, width), -1, dtype=torch.int32), 0
    for b, h in enumerate(held):
        table[b, :h] = torch.tensor(order[at:at + h], dtype=torch.int32)
        at += h
    ring = [-9] * size
    for i in range(free):
        ring[(head + i) % size] = order[used + i]
    new, want, want_ring = [], table.clone(), list(ring)
    wanted = back = taken = given = 0
    for b, (n, d) in enumerate(zip(lens, delta)):
        to = max(0, n + d)
        have, then = held[b], -(-to // page)
        wanted, back = wanted + max(0, then - have), back + max(0, have - then)
        if (then > have and wanted > free) or (then < have and back > size - free):
            to = n
        for p in range(have, -(-to // page)):
            want[b, p] = ring[(head + taken) % size]
            taken += 1
        for p in range(-(-to // page), have):
            want_ring[(head + free + given) % size] = int(table[b, p])
            given += 1
        new.append(to)
    d_table, d_ring, err = table.cuda(), dev(ring), err_word()
    capacity = sum(max(0, n - m) for n, m in zip(new, lens))
    t = D.advance_tables(dev(lens), dev(delta), d_table, d_ring, dev([head, head + free], torch.int64), page, capacity, err)
    assert int(err.item()) == (5 if back > size - free else 0)
    assert t.lens.tolist() == new and t.counters.tolist() == [head + taken, head + free + given]
    assert d_ring.tolist() == want_ring and torch.equal(d_table.cpu(), want)
    pos = t.positions.tolist()
    assert t.slots.tolist() == [int(want[b, p // page]) * page + p % page for b, p in zip(t.rows.tolist(), pos)]
    assert pos == [p for n, m in zip(lens, new) for p in range(n, m)]


@pytest.mark.parametrize("bad", [-1, -9, -2 ** 31, 2 ** 27, 2 ** 31 - 1])
def test_advance_tables_page_ids_out_of_range(D, bad):
    """They are recorded, passed on as -1 and never become another page's slot. 2^27 pages of 16 are beyond 32-bit slots."""
    # an append into a page that the table does not have, and one that takes a bad entry of the ring
    table, ring, err = dev([[bad, 7, 7], [1, 7, 7]]), dev([bad, 4, -5, -5, -5]), err_word()
    t = D.advance_tables(dev([10, 16]), dev([3, 20]), table, ring, dev([0, 2], torch.int64), 16, 30, err)
    assert int(err.item()) == 6
    assert t.lens.tolist() == [13, 36] and t.counters.tolist() == [2, 2] and t.cu.tolist() == [0, 3, 23]
    assert t.slots.tolist() == [-1] * 3 + [-1] * 16 + [64 + i for i in range(4)] + [-1] * 7
    assert t.positions.tolist() == list(range(10, 13)) + list(range(16, 36)) + [-1] * 7
    assert table.tolist() == [[bad, 7, 7], [1, -1, 4]] and ring.tolist() == [bad, 4, -5, -5, -5]
    # pages given back
    table, ring, err = dev([[3, bad, 2], [bad, 7, 7]]), dev([-5] * 5), err_word()
    t = D.advance_tables(dev([40, 1]), dev([-40, 0]), table, ring, dev([5, 5], torch.int64), 16, 0, err)
    assert int(err.item()) == 6
    assert t.lens.tolist() == [0, 1] and t.counters.tolist() == [5, 8] and ring.tolist() == [3, -1, 2, -5, -5]
    # the largest id there is
    top = 2 ** 27 - 1
    err = err_word()
    t = D.advance_tables(dev([14]), dev([2]), dev([[top]]), dev([0]), dev([0, 0], torch.int64), 16, 2, err)
    assert int(err.item()) == 0 and t.slots.tolist() == [2 ** 31 - 2, 2 ** 31 - 1]


def test_advance_tables_page_ids_out_of_range_in_long_lists(D):
    """Four tokens a thread."""
    rows, page, width = 512, 16, 130
    table = torch.arange(rows * width, dtype=torch.int32).view(rows, width)
    table[5, 0], table[77, 0], table[400, 0] = -3, 2 ** 30, -1
    d_table, err = table.cuda(), err_word()
    ring = torch.arange(10 ** 6, 10 ** 6 + rows * 125, dtype=torch.int32)
    ring[17], ring[40000] = -4, 2 ** 27
    d_ring = torch.cat([ring, torch.full((rows,), -5, dtype=torch.int32)]).cuda()
    t = D.advance_tables(dev([3] * rows), dev([2000] * rows), d_table, d_ring, dev([0, len(ring)], torch.int64), page,
                         2000 * rows + 5, err)
    assert int(err.item()) == 6 and t.lens.tolist() == [2003] * rows
    ring = torch.where((ring < 0) | (ring >= 2 ** 27), torch.tensor(-1, dtype=torch.int32), ring)
    want = table.clone()
    want[:, 1:126] = ring.view(rows, 125)
    assert torch.equal(d_table.cpu(), want)
    pos = torch.arange(3, 2003)
    ids = want.long()[:, pos // page]
    slots = torch.where((ids < 0) | (ids >= 2 ** 27), torch.tensor(-1), ids * page + pos % page)
    assert torch.equal(t.slots.cpu(), torch.cat([slots.flatten(), torch.full((5,), -1)]).to(torch.int32))


# ---- tokens that no request claims, and requests that are refused ---------------------------------------------------
def dirty(*shape, dtype):
    """Leaves memory of NaN for the next allocation of this size."""
    x = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
    y = torch.full(shape[:2], float("nan"), device="cuda")
    del x, y


def blank(out, lse):
    return bool((out == 0).all()) and bool((lse == float("-inf")).all())


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_tree_attention_tokens_of_no_request(D, dim):
    """A buffer longer than the requests' tokens (a fixed size in a graph): what lies around them is 0 and -inf, no error."""
    c = Case([300, 0, 2000], [4, 3, 9], 8, 2, dim, 16, F16, seed=3)
    out, lse = c.check(D)
    lead, trail = 5, 1000
    pad = lambda x: torch.cat([x.new_full((lead, *x.shape[1:]), 7), x, x.new_full((trail, *x.shape[1:]), 7)])  # noqa: E731
    c.q, c.k, c.v, c.mask, c.positions = (pad(x) for x in (c.q, c.k, c.v, c.mask, c.positions))
    c.cu = [lead + x for x in c.cu]
    dirty(*c.q.shape, dtype=F16)
    err = err_word()
    more, more_lse = c.call(D, err=err)
    assert int(err.item()) == 0
    mine = slice(lead, lead + len(out))
    assert torch.equal(more[mine], out) and torch.equal(more_lse[mine], lse)
    assert blank(more[:lead], more_lse[:lead]) and blank(more[-trail:], more_lse[-trail:])


def test_tree_attention_without_requests(D):
    c = Case([40], [6], 8, 2, 128, 16, F16, seed=3)
    c.lens, c.cu, c.table = [], [0], c.table[:0]
    dirty(*c.q.shape, dtype=F16)
    assert blank(*c.call(D))


@pytest.mark.parametrize("lens,cu,max_tree,refused", [
    ([100, -1, 50], [0, 4, 9, 12], 16, [(4, 9)]), ([100, 10 ** 6, 50], [0, 4, 9, 12], 16, [(4, 9)]),
    ([100, 60, 50], [0, 4, 9, 12], 4, [(4, 9)]), ([100, 60, 50], [0, 4, 9, 14], 16, [(9, 12)]),
    ([100, 60, 50], [-2, 4, 9, 12], 16, [(0, 4)]), ([-5, -5, -5], [1, 4, 4, 12], 16, [(0, 12)])])
def test_tree_attention_refused_requests_see_nothing(D, lens, cu, max_tree, refused):
    """The others are what they are without them."""
    c = Case([100, 60, 50], [4, 5, 3], 8, 2, 128, 16, F16, seed=4, max_tree=16)
    out, lse = c.check(D)
    c.lens, c.cu, c.max_tree = lens, cu, max_tree
    dirty(*c.q.shape, dtype=F16)
    err = err_word()
    got, got_lse = c.call(D, err=err)
    assert int(err.item()) == 5
    rest = torch.ones(12, dtype=torch.bool)
    for a, b in refused:
        assert blank(got[a:b], got_lse[a:b])
        rest[a:b] = False
    rest = rest.cuda()
    assert torch.equal(got[rest], out[rest]) and torch.equal(got_lse[rest], lse[rest])


@pytest.mark.parametrize("cu,max_tree,refused,code", [
    ([3, 5, 9], 64, [], 0), ([0, 5, 9], 64, [], 0), ([3, 5, 40], 32, [(5, 40)], 5), ([-1, 5, 9], 64, [(0, 5)], 5),
    ([0, 40, 90], 64, [(40, 60)], 5)])
def test_plan_tree_tokens_of_no_request(D, cu, max_tree, refused, code):
    """They, and those of refused requests, have position -1 and no bits."""
    tokens, words = 60, (max_tree + 31) // 32
    parents = dev([-1] * tokens)
    torch.full((tokens,), 77, dtype=torch.int32, device="cuda"), torch.full((tokens, words), 77, dtype=torch.int32, device="cuda")
    err = err_word()
    positions, mask = D.plan_tree(parents, dev(cu), dev([10, 20]), max_tree, err)
    assert int(err.item()) == code
    want = torch.full((tokens,), -1, dtype=torch.int32)
    bits = torch.zeros(tokens, words, dtype=torch.int64)
    for b in range(2):
        for t in range(max(cu[b], 0), min(cu[b + 1], tokens)):
            if not any(x <= t < y for x, y in refused):
                want[t] = (10, 20)[b]
                bits[t, (t - cu[b]) // 32] = 1 << (t - cu[b]) % 32
    bits = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
    assert torch.equal(positions.cpu(), want) and torch.equal(mask.cpu(), bits)


def test_plan_tree_without_requests(D):
    torch.full((6,), 77, dtype=torch.int32, device="cuda")
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    positions, mask = D.plan_tree(dev([-1] * 6), dev([0]), e, 4)
    assert positions.tolist() == [-1] * 6 and not bool(mask.any())


# ---- a cache used on several streams --------------------------------------------------------------------------------
def test_cache_attends_on_two_streams_at_once(D):
    """Items that are cut leave partial results in a workspace: calls that overlap must not share one."""
    layers, rows, page, hq, hkv, dim, n = 2, 3, 16, 16, 4, 128, 5
    cache = D.DraftCache(layers, rows, 3000, page, 16000, hkv, dim, BF16)
    cache.advance(dev([15000, 9000, 12001]), 0)
    g = torch.Generator(device="cuda").manual_seed(2)
    for x in (cache.k, cache.v):
        x.normal_(generator=g)
    cu = dev([0, n, 2 * n, 3 * n])
    new = [[torch.randn(3 * n, h, dim, generator=g, device="cuda").to(BF16) for h in (hq, hkv, hkv)] for _ in range(layers)]
    want = [cache.attend(layer, *new[layer], cu, 0.09, n) for layer in range(layers)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(layers)]
    got = []
    for _ in range(40):
        for layer, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append((layer, cache.attend(layer, *new[layer], cu, 0.09, n)))
    torch.cuda.synchronize()
    for layer, (out, lse) in got:
        assert torch.equal(out, want[layer][0]) and torch.equal(lse, want[layer][1])
    cache.err.zero_()  # advance listed none of its tokens


# ---- autograd -------------------------------------------------------------------------------------------------------
def test_inputs_that_want_gradients_are_refused(D):
    """There are no backward passes: such a call must not lose a gradient in silence."""
    c = Case([40], [3], 8, 2, 128, 16, F16, seed=1)
    w, inv = torch.ones(128, device="cuda"), torch.ones(32, device="cuda")
    learned = torch.nn.Parameter(torch.ones(128, device="cuda"))

    def norm(weight):
        return D.norm_rope(c.q, c.k, c.v, weight, w, inv, c.positions, 1e-6, F16)

    want = norm(w)
    with pytest.raises(ValueError, match="gradient"):
        norm(learned)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(norm(learned), want))
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(norm(learned), want))
    plain = c.call(D)
    c.q = c.q.detach().requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        c.call(D)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(c.call(D), plain))
    with pytest.raises(ValueError, match="gradient"):
        D.store_rows(c.k.detach().requires_grad_(), c.v, c.kc, c.vc, dev([0, 1, 2]))


def test_what_changes_in_place_says_so(D):
    """autograd, and others that compare version counters, see the change."""
    c = Case([40], [3], 8, 2, 128, 16, F16, seed=1)
    before = c.kc._version, c.vc._version
    D.store_rows(c.k, c.v, c.kc, c.vc, dev([0, 1, 2]))
    assert c.kc._version > before[0] and c.vc._version > before[1]
    w, inv, before = torch.ones(128, device="cuda"), torch.ones(32, device="cuda"), (c.kc._version, c.vc._version)
    D.norm_rope_store(c.q, c.k, c.v, w, w, inv, c.positions, 1e-6, c.kc, c.vc, dev([0, 1, 2]))
    assert c.kc._version > before[0] and c.vc._version > before[1]
    table, ring = dev([[0, -1]]), dev([1, 2])
    before = table._version, ring._version
    D.advance_tables(dev([16]), dev([1]), table, ring, dev([0, 2], torch.int64), 16, 1)
    assert table._version > before[0] and ring._version > before[1]
    with torch.inference_mode():
        cache = torch.zeros(2, 16, 2, 128, device="cuda", dtype=F16)
    D.store_rows(c.k, c.v, cache, cache.clone(), dev([0, 1, 2]))  # without a version counter
    assert torch.equal(cache[0, :3], c.k)


# ---- arguments and storage ------------------------------------------------------------------------------------------
def test_numpy_integers_are_integers(D):
    parents, cu, lens = dev([-1, 0]), dev([0, 2]), dev([5])
    for kind in (np.int32, np.int64, np.uint8):
        positions, _ = D.plan_tree(parents, cu, lens, kind(2))
        assert positions.tolist() == [5, 6]
    for wrong in (np.float32(2), torch.tensor(2), torch.tensor(2, device="cuda"), 2.0, "2", None, np.int64(0), np.int64(1 << 40)):
        with pytest.raises(ValueError):
            D.plan_tree(parents, cu, lens, wrong)


def test_lengths_do_not_keep_the_lists(D):
    """What a cache keeps from call to call (lengths, counters) shares no memory with the lists of a call's tokens."""
    t = D.advance_tables(dev([0, 3]), dev([1000, 2]), dev([[-1] * 70, [0] + [-1] * 69]), dev(list(range(1, 101))),
                         dev([0, 100], torch.int64), 16, 100000)
    assert t.lens.tolist() == [1000, 5] and t.counters.tolist() == [63, 100] and t.cu.tolist() == [0, 1000, 1002]
    assert t.slots.shape == t.rows.shape == t.positions.shape == (100000,)
    for kept in (t.lens, t.counters, t.cu):
        assert kept.untyped_storage().nbytes() < 4096
    assert t.counters.dtype == torch.int64 and t.lens.is_contiguous() and t.cu.is_contiguous()


@pytest.mark.parametrize("device", [None, 0, "cuda", "cuda:0", torch.device("cuda"), torch.device("cuda", 0)])
def test_cache_devices(D, device):
    cache = D.DraftCache(1, 2, 4, 8, 16, 1, 64, device=device)
    assert {x.device for x in (cache.k, cache.table, cache.lens, cache.counters, cache.err)} == {torch.device("cuda", 0)}
    cache.advance(dev([3, 9]), 12)
    assert cache.lens.tolist() == [3, 9]
    with pytest.raises(ValueError):
        D.DraftCache(1, 2, 4, 8, 16, 1, 64, device="cpu")


def test_the_next_tick_waits_for_reads_of_the_rings(weights_seed0):
    """Attention that is still queued when the engine's next tick is called reads the rings as they were."""
    from hs_guard_b200 import drafts
    from hs_guard_b200.engine import SlotEngine
    eng = SlotEngine(weights_seed0, 2)
    rng = np.random.default_rng(9)
    eng.step([(s, rng.integers(0, 1000, 600).tolist()) for s in range(2)])
    k_cache, v_cache, table, lens = drafts.ring_cache(eng, 4, [0, 1])
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(6, h, 256, generator=g, device="cuda").half() for h in (8, 2, 2))
    cu = torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda")

    def attend():
        return drafts.tree_attention(q, k, v, k_cache, v_cache, table, lens, cu, 1.0 / 16, 3, window=512)

    want, want_lse = attend()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # a tenth of a second: the tick would be through long before
        out, lse = attend()
        drafts.ring_done(eng)
    eng.step([(s, rng.integers(0, 1000, 64).tolist()) for s in range(2)])
    assert side.query()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    assert not torch.equal(attend()[0], want)  # the rings have moved on
    torch.cuda.synchronize()
    eng.close()


# ---- the widest shapes ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lens,counts,hq,hkv,dim,page,dtype,window", [
    ([300, 31], [3, 2], 128, 1, 64, 16, F16, 0), ([129], [5], 128, 1, 128, 16, BF16, 0), ([70, 600], [2, 3], 256, 2, 256, 16, F16, 200),
    ([200, 9], [4, 7], 100, 1, 64, 8, BF16, 0), ([1000], [3], 65, 1, 128, 32, F16, 0), ([257, 40], [9, 4], 66, 2, 64, 16, F16, 30),
    ([500], [11], 24, 1, 256, 48, BF16, 0), ([50, 0, 700], [1, 6, 2], 33, 3, 128, 16, F16, 0)])
def test_tree_attention_many_query_heads_a_key_head(D, lens, counts, hq, hkv, dim, page, dtype, window):
    """Groups of 11 to 128 query heads, most of which leave rows of a block without a token."""
    Case(lens, counts, hq, hkv, dim, page, dtype, window, seed=hq).check(D)


@pytest.mark.parametrize("mask,window", [("tree", 0), ("holes", 0), (None, 0), ("tree", 300), (None, 300)])
def test_tree_attention_largest_trees(D, mask, window):
    """1,024 drafted tokens: all 32 mask words, drafts of many tiles, and windows that end among them."""
    Case([90, 700], [1024, 1000], 2, 1, 64, 16, F16, window, mask=mask, seed=5).check(D)


@pytest.mark.parametrize("tokens", [1, 37])
def test_norm_rope_is_the_models(D, tokens):
    """The classifier's own norm and rotation (32-bit, written for the oracle) of its fused projection, at positions where a
    32-bit angle is exact enough: 4,000 x 2^-24 x |y| below an fp16 result's rounding."""
    from hs_guard_b200 import DEFAULT as cfg
    from oracle import stream
    g = torch.Generator().manual_seed(tokens)
    hq, hkv, dim, rot = cfg.attn_heads, cfg.kv_heads, cfg.attn_head_dim, cfg.rotary_dim
    proj = torch.randn(tokens, (2 * hq + 2 * hkv) * dim, generator=g)
    q = proj[:, :2 * hq * dim].view(tokens, hq, 2 * dim)[..., :dim]
    k = proj[:, 2 * hq * dim:(2 * hq + hkv) * dim].view(tokens, hkv, dim)
    v = proj[:, (2 * hq + hkv) * dim:].view(tokens, hkv, dim)
    wq, wk = (1 + 0.2 * torch.randn(dim, generator=g) for _ in range(2))
    inv = 1.0 / cfg.rope_theta ** (torch.arange(0, rot, 2, dtype=torch.int64).float() / rot)
    pos = torch.randint(0, 4000, (tokens,), generator=g)
    angle = torch.cat([pos[:, None].float() * inv] * 2, -1)
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    gq, gk, gv = D.norm_rope(*(x.cuda() for x in (q, k, v, wq, wk, inv)), dev(pos), cfg.rms_eps, F16)
    for got, x, w in ((gq, q, wq), (gk, k, wk)):
        ref = stream.rope(stream.rms_norm(x, w, cfg.rms_eps), cos, sin, rot)
        tol = U[F16] * ref.abs() + (1e-5 + 4000 * 2.0 ** -24) * ref.abs().amax(-1, keepdim=True) + TINY[F16]
        assert bool(((got.cpu() - ref).abs() <= tol).all())
    assert torch.equal(gv.cpu(), v.half())
