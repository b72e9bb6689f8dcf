"""Draft scoring operators (hs_guard_b200.drafts) on a B200 against plain 64-bit implementations.

Tolerances, with u the result type's unit roundoff (2^-11 fp16, 2^-8 bf16):
  norm and rotation   u |y| for the result's rounding + 1e-5 of the row's largest |y| for the fp32 arithmetic (a sum of
                      256 squares and a handful of products: below 40 roundings of 2^-24) + the smallest subnormal
  attention           u |o| for the result's rounding + (u + 2 ds) sum_n p_n |v_n|: u for the softmax weights, which
                      enter the second product in the result's type, and ds = dim 2^-24 scale max |q| |k| for the
                      fp32 sum of the scores (a weight's relative error is at most twice its score's absolute one)
  log-sum-exp         ds + 4e-6 (1 + |lse|): exponentials to 2^-22 and the sum's and logarithm's rounding
Integers, and rows copied by store_rows, are equal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -134}


@pytest.fixture(scope="module")
def D():
    from hs_guard_b200.build import build
    build()
    from hs_guard_b200 import drafts
    return drafts


def dev(x, dtype=torch.int32):
    return torch.as_tensor(x, dtype=dtype).cuda()


def err_word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


# ---- advance_tables -------------------------------------------------------------------------------------------------
def tables_reference(lens, delta, table, ring, head, tail, page):
    """One request after another, over Python lists (changed in place)."""
    width, size, avail = len(table[0]), len(ring), tail - head
    new, listed, wanted, taken, given = [], [], 0, 0, 0
    for b, (n, d) in enumerate(zip(lens, delta)):
        to = max(0, n + d)
        have, want = -(-n // page), -(-to // page)
        if to > width * page:
            new.append(n)
            listed.append(0)
            continue
        wanted += max(0, want - have)
        if want > have and wanted > avail:
            new.append(n)
            listed.append(0)
            continue
        for p in range(have, want):
            table[b][p] = ring[(head + taken) % size]
            taken += 1
        for p in range(want, have):
            ring[(tail + given) % size] = table[b][p]
            given += 1
        new.append(to)
        listed.append(max(0, to - n))
    cu = [0]
    for c in listed:
        cu.append(cu[-1] + c)
    tokens = [(table[b][p // page] * page + p % page, b, p) for b, c in enumerate(listed)
              for p in range(lens[b], lens[b] + c)]
    return new, [head + taken, tail + given], cu, tokens


@pytest.mark.parametrize("rows,page,top,grow,free_share,pad", [
    (1, 16, 0, 1, 1.0, 0), (1, 8, 40, 1, 1.0, 3), (7, 16, 100, 40, 1.0, 5), (7, 16, 100, 40, 0.5, 0),
    (352, 64, 2000, 6, 1.0, 1), (1025, 24, 300, 90, 0.8, 2), (4096, 16, 50, 3, 0.9, 7), (33, 1, 20, 9, 0.7, 4),
    (64, 128, 5000, 4000, 0.6, 0)])
def test_advance_tables(D, rows, page, top, grow, free_share, pad):
    g = torch.Generator().manual_seed(rows * 31 + page)
    lens = torch.randint(0, top + 1, (rows,), generator=g).tolist()
    delta = torch.randint(-grow, grow + 1, (rows,), generator=g).tolist()
    if rows > 4:
        delta[1], delta[2], delta[3] = 0, -10 ** 6, 10 ** 8  # nothing, everything back, past the table's width
    width = -(-(top + grow) // page) + 1
    held = [-(-n // page) for n in lens]
    want = sum(max(0, -(-(n + d) // page) - h) for n, d, h in zip(lens, delta, held) if n + d <= width * page)
    free = int(want * free_share) + (2 if free_share == 1.0 else 0)
    pages = sum(held) + free
    pages = max(pages, 1)
    order = torch.randperm(pages, generator=g).tolist()
    table, at = [], 0
    for h in held:
        table.append(order[at:at + h] + [-7] * (width - h))
        at += h
    head = 3 * pages + pages // 2
    ring = [-9] * pages
    for i in range(free):
        ring[(head + i) % pages] = order[at + i]
    wide = torch.full((rows, width + pad), -5, dtype=torch.int32, device="cuda")
    d_table = wide[:, :width]
    d_table.copy_(dev(table))
    d_ring, d_lens, d_delta = dev(ring), dev(lens), dev(delta)
    counters = dev([head, head + free], torch.int64)
    new, new_counters, cu, tokens = tables_reference(lens, delta, table, ring, head, head + free, page)
    capacity = len(tokens) + pad
    err = err_word()
    for _ in range(2):  # the same call again gives the same result
        t = D.advance_tables(d_lens, d_delta, d_table, d_ring, counters, page, capacity, err)
        assert int(err.item()) == 0
        assert t.lens.tolist() == new and t.counters.tolist() == new_counters and t.cu.tolist() == cu
        none = [(-1, -1, -1)] * pad
        assert list(zip(t.slots.tolist(), t.rows.tolist(), t.positions.tolist())) == tokens + none
        assert d_table.tolist() == table and d_ring.tolist() == ring
    assert torch.all(wide[:, width:] == -5)
    assert d_lens.tolist() == lens and counters.tolist() == [head, head + free]


def test_advance_tables_no_requests_and_short_capacity(D):
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    t = D.advance_tables(empty, empty, torch.empty(0, 4, dtype=torch.int32, device="cuda"), dev([3, 4]),
                         dev([0, 2], torch.int64), 16, 3)
    assert t.cu.tolist() == [0] and t.counters.tolist() == [0, 2] and t.slots.tolist() == [-1] * 3
    err = err_word()
    t = D.advance_tables(dev([0, 5]), dev([10, 20]), dev([[-1, -1], [1, -1]]), dev([2, 3, 0, 4]),
                         dev([0, 2], torch.int64), 16, 12, err)
    assert t.slots.tolist() == [32 + i for i in range(10)] + [16 + 5, 16 + 6] and t.cu.tolist() == [0, 10, 30]
    assert int(err.item()) == 5
    with pytest.raises(RuntimeError, match="length"):
        D.raise_device_error(err)
    assert int(err.item()) == 0


def test_advance_tables_records_a_bad_length(D):
    err = err_word()
    t = D.advance_tables(dev([40, 3, -2]), dev([1, 1, 1]), dev([[0, 1], [2, -1], [-1, -1]]), dev([5, 6]),
                         dev([0, 2], torch.int64), 16, 4, err)
    assert int(err.item()) == 5
    assert t.lens.tolist() == [40, 4, -2] and t.slots.tolist() == [35, -1, -1, -1] and t.counters.tolist() == [0, 2]


# ---- plan_tree ------------------------------------------------------------------------------------------------------
def random_parents(counts, g, chain=False):
    out = []
    for n in counts:
        for i in range(n):
            out.append(i - 1 if chain else int(torch.randint(-1, max(i, 1), (1,), generator=g)) if i else -1)
    return out


def tree_reference(parents, counts):
    masks, depths, at = [], [], 0
    for n in counts:
        m, d = [], []
        for i in range(n):
            p = parents[at + i]
            m.append((m[p] if p >= 0 else 0) | 1 << i)
            d.append(d[p] + 1 if p >= 0 else 0)
        masks += m
        depths += d
        at += n
    return masks, depths


def pack_masks(masks, words):
    vals = [[(m >> 32 * w) & 0xffffffff for w in range(words)] for m in masks]
    t = torch.tensor(vals, dtype=torch.int64).reshape(len(masks), words)
    return torch.where(t >= 1 << 31, t - (1 << 32), t).to(torch.int32)


@pytest.mark.parametrize("counts,chain,max_tree", [
    ([1], False, 1), ([15], False, 15), ([0, 3, 0, 64, 33], False, 64), ([1024, 5], True, 1024),
    ([200] * 40, False, 200), ([31, 32, 1], True, 97)])
def test_plan_tree(D, counts, chain, max_tree):
    g = torch.Generator().manual_seed(len(counts) + max_tree)
    parents = random_parents(counts, g, chain)
    lens = torch.randint(0, 1000, (len(counts),), generator=g).tolist()
    masks, depths = tree_reference(parents, counts)
    cu = [0] + torch.cumsum(torch.tensor(counts), 0).tolist()
    err = err_word()
    positions, mask = D.plan_tree(dev(parents), dev(cu), dev(lens), max_tree, err)
    assert int(err.item()) == 0
    assert torch.equal(mask.cpu(), pack_masks(masks, (max_tree + 31) // 32))
    assert positions.tolist() == [lens[b] + d for b, n in enumerate(counts)
                                  for d in depths[cu[b]:cu[b] + n]]


@pytest.mark.parametrize("parents", [[-1, 1], [-1, 5], [-2, 0]])
def test_plan_tree_records_a_bad_parent(D, parents):
    err = err_word()
    D.plan_tree(dev(parents), dev([0, 2]), dev([4]), 2, err)
    assert int(err.item()) == 7


# ---- norm_rope ------------------------------------------------------------------------------------------------------
def norm_reference(x, w, inv, pos, eps):
    x, r = x.double(), inv.shape[0]
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    a = (pos.double()[:, None] * inv.double())[:, None]
    lo, hi = y[..., :r].clone(), y[..., r:2 * r].clone()
    y[..., :r] = lo * torch.cos(a) - hi * torch.sin(a)
    y[..., r:2 * r] = hi * torch.cos(a) + lo * torch.sin(a)
    return y


def close_rows(got, ref, dtype):
    tol = U[dtype] * ref.abs() + 1e-5 * ref.abs().amax(-1, keepdim=True) + TINY[dtype]
    assert torch.all((got.double().cpu() - ref.cpu()).abs() <= tol.cpu())


@pytest.mark.parametrize("tokens,hq,hkv,dim,rot,tin,tout", [
    (1, 8, 2, 256, 64, F32, F16), (5, 8, 2, 256, 256, F32, BF16), (17, 15, 5, 64, 64, BF16, BF16),
    (300, 7, 1, 128, 32, F16, F16), (33, 1, 1, 64, 16, F16, BF16), (9, 3, 3, 128, 112, BF16, F16),
    (2049, 6, 2, 128, 128, BF16, BF16)])
@pytest.mark.parametrize("gate", [False, True])
def test_norm_rope(D, tokens, hq, hkv, dim, rot, tin, tout, gate):
    g = torch.Generator(device="cuda").manual_seed(tokens + dim)
    step = 2 * dim if gate else dim
    x = torch.randn(tokens, hq * step + 2 * hkv * dim, generator=g, device="cuda").to(tin)
    q = x[:, :hq * step].view(tokens, hq, step)[:, :, :dim]
    k = x[:, hq * step:hq * step + hkv * dim].view(tokens, hkv, dim)
    v = x[:, hq * step + hkv * dim:].view(tokens, hkv, dim)
    q[0, 0] = 0  # a row of zeros stays zero
    wq, wk = torch.randn(dim, generator=g, device="cuda"), torch.randn(dim, generator=g, device="cuda")
    inv = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda").float() / rot)
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda").to(torch.int32)
    pos[-1] = (1 << 24) + 77777  # no longer an fp32 integer
    gq, gk, gv = D.norm_rope(q, k, v, wq, wk, inv, pos, 1e-6, tout)
    assert gq.dtype == gk.dtype == gv.dtype == tout and gq.is_contiguous() and gk.is_contiguous()
    close_rows(gq, norm_reference(q, wq, inv, pos, 1e-6), tout)
    close_rows(gk, norm_reference(k, wk, inv, pos, 1e-6), tout)
    assert torch.equal(gv, v.to(tout))


@pytest.mark.parametrize("heads_first", [False, True])
def test_norm_rope_store_writes_its_slots_only(D, heads_first):
    tokens, hq, hkv, dim, page = 41, 4, 2, 128, 24
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(tokens, h, dim, generator=g, device="cuda") for h in (hq, hkv, hkv))
    w, inv = torch.ones(dim, device="cuda"), 10000.0 ** (-torch.arange(0, 64, 2, device="cuda").float() / 64)
    pos = torch.arange(tokens, device="cuda", dtype=torch.int32)
    shape = (5, hkv, page, dim) if heads_first else (5, page, hkv, dim)
    kc, vc = (torch.full(shape, 9.0, device="cuda", dtype=BF16) for _ in range(2))
    if heads_first:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    slots = torch.randperm(5 * page, generator=torch.Generator().manual_seed(1))[:tokens].to(torch.int32).cuda()
    slots[7] = -1
    slots[8] = 5 * page  # beyond the pages: skipped and recorded
    err = err_word()
    gq = D.norm_rope_store(q, k, v, w, w, inv, pos, 1e-6, kc, vc, slots, err)
    assert int(err.item()) == 3
    rq, rk, rv = D.norm_rope(q, k, v, w, w, inv, pos, 1e-6, BF16)
    assert torch.equal(gq, rq)
    want_k, want_v = torch.full((5 * page, hkv, dim), 9.0, dtype=BF16), torch.full((5 * page, hkv, dim), 9.0, dtype=BF16)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < 5 * page:
            want_k[s], want_v[s] = rk[t].cpu(), rv[t].cpu()
    assert torch.equal(kc.reshape(-1, hkv, dim).cpu(), want_k) and torch.equal(vc.reshape(-1, hkv, dim).cpu(), want_v)


# ---- tree_attention -------------------------------------------------------------------------------------------------
class Case:
    """Inputs of one tree_attention call and their 64-bit result, request by request."""

    def __init__(self, lens, counts, hq, hkv, dim, page, dtype, window=0, heads_first=False, mask="tree", seed=0,
                 spread=1.0, junk=float("nan"), max_tree=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        cg = torch.Generator().manual_seed(seed)
        self.lens, self.counts, self.dim, self.window, self.dtype, self.group = lens, counts, dim, window, dtype, hq // hkv
        self.hq, self.hkv, self.page = hq, hkv, page
        total = sum(counts)
        self.max_tree = max_tree or max(1, max(counts))
        held = [-(-n // page) for n in lens]
        pages = sum(held) + 3
        order = torch.randperm(pages, generator=cg)
        width = max(1, max(held))
        table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
        for b, h in enumerate(held):
            table[b, :h] = order[at:at + h].to(torch.int32)
            at += h
            if window:  # given back: never read
                table[b, :max(0, lens[b] - window + 1) // page] = 1 << 30
        self.table = table.cuda()
        shape = (pages, hkv, page, dim) if heads_first else (pages, page, hkv, dim)
        self.kc, self.vc = (torch.randn(shape, generator=g, device="cuda").mul(spread).to(dtype) for _ in range(2))
        if heads_first:
            self.kc, self.vc = self.kc.transpose(1, 2), self.vc.transpose(1, 2)
        for b, n in enumerate(lens):
            if n % page:
                last = int(self.table[b, n // page])
                self.kc[last, n % page:], self.vc[last, n % page:] = junk, junk
        self.kc[order[-3:]], self.vc[order[-3:]] = junk, junk
        # q, k and v as slices of one projection
        width_x = (hq + 2 * hkv) * dim + 24
        x = torch.randn(max(total, 1), width_x, generator=g, device="cuda").mul(spread).to(dtype)[:total]
        self.q = x[:, :hq * dim].unflatten(1, (hq, dim))
        self.k = x[:, hq * dim:(hq + hkv) * dim].unflatten(1, (hkv, dim))
        self.v = x[:, (hq + hkv) * dim:(hq + 2 * hkv) * dim].unflatten(1, (hkv, dim))
        self.cu = [0] + torch.cumsum(torch.tensor(counts), 0).tolist()
        words = (self.max_tree + 31) // 32
        parents = random_parents(counts, cg, chain=mask is None)
        masks, depths = tree_reference(parents, counts)
        if mask == "holes":  # any bits: tokens that see no drafted one, themselves included, among them
            masks = [0 if i % 3 == 0 else m ^ (m & 0x55) for i, m in enumerate(masks)]
        self.bits = masks
        self.mask = None if mask is None else pack_masks(masks, words).cuda()
        row = [b for b, n in enumerate(counts) for _ in range(n)]
        self.positions = dev([lens[b] + d for b, d in zip(row, depths)]) if total else torch.empty(
            0, dtype=torch.int32, device="cuda")
        self.scale = 1.0 / math.sqrt(dim)

    def call(self, D, **more):
        args = dict(mask=self.mask, positions=self.positions, window=self.window)
        args.update(more)
        return D.tree_attention(self.q, self.k, self.v, self.kc, self.vc, self.table, dev(self.lens), dev(self.cu),
                                self.scale, self.max_tree, **args)

    def reference(self):
        """(out, lse, tolerance of out, tolerance of lse)"""
        outs, lses, tols, ltols = [], [], [], []
        pos = self.positions.tolist()
        for b, n in enumerate(self.lens):
            t0, t1 = self.cu[b], self.cu[b + 1]
            if t0 == t1:
                continue
            start = max(0, n - self.window + 1) if self.window else 0
            at = torch.arange(start, n, device="cuda")
            pages = self.table[b][at // self.page].long()
            old_k, old_v = self.kc[pages, at % self.page].double(), self.vc[pages, at % self.page].double()
            for t in range(t0, t1):
                low = pos[t] - self.window if self.window else -1
                keep = at > low
                js = [j for j in range(t1 - t0) if (self.bits[t] >> j & 1 if self.mask is not None else j <= t - t0)
                      and (pos[t0 + j] > low)]
                k = torch.cat([old_k[keep], self.k[t0:t1][js].double()])
                v = torch.cat([old_v[keep], self.v[t0:t1][js].double()])
                q = self.q[t].double().view(self.hkv, self.group, self.dim)
                s = torch.einsum("hgd,nhd->hgn", q, k) * self.scale
                if s.shape[-1] == 0:
                    outs.append(torch.zeros(self.hq, self.dim, dtype=torch.float64, device="cuda"))
                    lses.append(torch.full((self.hq,), float("-inf"), dtype=torch.float64, device="cuda"))
                    tols.append(torch.zeros_like(outs[-1]))
                    ltols.append(torch.zeros_like(lses[-1]))
                    continue
                p = torch.softmax(s, -1)
                o = torch.einsum("hgn,nhd->hgd", p, v)
                ds = self.dim * 2.0 ** -24 * self.scale * float(q.norm(dim=-1).max() * k.norm(dim=-1).max())
                u = U[self.dtype]
                lse = torch.logsumexp(s, -1)
                tols.append((u * o.abs() + (u + 2 * ds) * torch.einsum("hgn,nhd->hgd", p, v.abs()) +
                             TINY[self.dtype]).reshape(self.hq, self.dim))
                outs.append(o.reshape(self.hq, self.dim))
                lses.append(lse.reshape(self.hq))
                ltols.append((ds + 4e-6 * (1 + lse.abs())).reshape(self.hq))
        return tuple(torch.stack(x) for x in (outs, lses, tols, ltols))

    def check(self, D, **more):
        err = err_word()
        out, lse = self.call(D, err=err, **more)
        assert int(err.item()) == 0
        ref, rlse, tol, ltol = self.reference()
        assert out.dtype == self.dtype and out.shape == ref.shape and lse.shape == rlse.shape
        bad = (out.double() - ref).abs() > tol
        assert not bool(bad.any() | out.isnan().any()), \
            f"{int(bad.sum())} of {bad.numel()} out of tolerance, worst {float(((out.double() - ref).abs() / tol.clamp(min=1e-30)).nan_to_num(1e9).max())}"
        both = (lse == float("-inf")) & (rlse == float("-inf"))
        assert torch.all(both | ((lse.double() - rlse).abs() <= ltol))
        return out, lse


SHAPES = [
    # lens, counts, hq, hkv, dim, page, dtype, window
    ([5], [1], 1, 1, 64, 16, F16, 0),
    ([0], [1], 8, 2, 256, 16, F16, 0),
    ([1, 0, 511, 512, 513], [1, 1, 1, 1, 1], 8, 2, 256, 16, F16, 0),
    ([700, 513, 0, 3000], [9, 1, 4, 0], 8, 2, 256, 16, F16, 512),
    ([127, 128, 129, 1000], [3, 7, 13, 2], 32, 8, 128, 64, BF16, 0),
    ([4000], [16], 4, 4, 128, 32, BF16, 0),
    ([333, 4097], [31, 64], 16, 2, 64, 8, BF16, 0),
    ([1000, 40], [65, 200], 7, 1, 128, 48, F16, 0),
    ([129, 2050], [40, 33], 32, 4, 256, 128, BF16, 0),
    ([2000, 10, 300], [20, 20, 20], 15, 5, 128, 24, BF16, 100),
    ([600, 7], [12, 12], 6, 2, 64, 256, F16, 3),
    ([90, 91], [5, 6], 8, 8, 64, 16, F16, 1),
    ([20000], [1], 8, 1, 128, 64, BF16, 0),
    ([3, 60000], [2, 5], 2, 1, 64, 40, F16, 0),
    ([128 * 9] * 30, [4] * 30, 16, 4, 128, 16, BF16, 0),
    ([17] * 600, [1] * 600, 2, 1, 64, 8, BF16, 0),
    ([50, 300], [300, 1], 4, 1, 128, 16, F16, 0),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[2]}x{s[3]}x{s[4]}p{s[5]}w{s[7]}n{len(s[0])}")
@pytest.mark.parametrize("mask,heads_first", [("tree", False), ("holes", True), (None, True)])
def test_tree_attention(D, shape, mask, heads_first):
    lens, counts, hq, hkv, dim, page, dtype, window = shape
    Case(lens, counts, hq, hkv, dim, page, dtype, window, heads_first, mask, seed=len(lens) + dim).check(D)


@pytest.mark.parametrize("spread", [1e-3, 4.0])
def test_tree_attention_flat_and_peaked_scores(D, spread):
    """Scores near zero (every key counts alike) and up to hundreds (one key decides; the running maximum moves)."""
    Case([1500, 37], [6, 11], 8, 2, 128, 16, BF16, spread=spread, seed=5).check(D)
    Case([1500, 37], [6, 11], 8, 2, 256, 16, F16, spread=min(spread, 3.0), seed=6).check(D)


@pytest.mark.parametrize("lens,counts,hq,hkv,dim,page,dtype,window", [
    ([1279], [1], 4, 1, 128, 16, BF16, 0), ([1281], [1], 4, 1, 128, 16, BF16, 0), ([639], [3], 2, 1, 256, 16, F16, 0),
    ([3845], [2], 16, 2, 64, 64, F16, 0), ([8000], [5], 2, 1, 128, 32, F16, 0), ([9001], [1], 8, 1, 256, 64, BF16, 0),
    ([14000, 0, 1], [1, 0, 2], 2, 1, 128, 48, BF16, 0), ([5, 9000, 300], [2, 70, 1], 4, 1, 128, 16, F16, 0),
    ([30000], [4], 3, 3, 64, 40, BF16, 20000)])
def test_tree_attention_pieces_of_few_long_items(D, lens, counts, hq, hkv, dim, page, dtype, window):
    """Few items of many tiles: a piece holds several of an item's tiles although more thread blocks are free, the last
    pieces of the line are empty, and an item's last part is shorter than the others."""
    Case(lens, counts, hq, hkv, dim, page, dtype, window, mask="holes" if dim == 64 else "tree", seed=sum(lens)).check(D)


def test_tree_attention_rising_scores(D):
    """Keys sorted so that the running maximum rises all along a long cache, by more than any fixed slack."""
    c = Case([3000], [2], 4, 1, 128, 8, F16, mask=None, seed=8)
    direction = torch.zeros(128, device="cuda")
    direction[0] = 1.0
    c.q[:] = (8 * direction).to(F16)
    at = torch.arange(3000, device="cuda")
    c.kc[c.table[0][at // 8].long(), at % 8, 0] = (torch.linspace(0, 60, 3000, device="cuda")[:, None] * direction).to(F16)
    c.check(D)


def test_tree_attention_what_is_not_seen_does_not_count(D):
    """NaN and infinities in other branches, in cached keys below some tokens' windows and past every length."""
    for window in (0, 40):
        c = Case([100, 200], [6, 5], 8, 2, 128, 16, F16, window=window, seed=11)
        clean, clean_lse = c.check(D)
        # drafted token 2 of request 0: itself and its descendants see it
        keep = [i for i in range(c.cu[1]) if not c.bits[i] >> 2 & 1]
        c.k[2], c.v[2] = float("nan"), float("inf")
        out, lse = c.call(D)
        assert torch.equal(out[keep], clean[keep]) and torch.equal(lse[keep], clean_lse[keep])
        assert torch.equal(out[c.cu[1]:], clean[c.cu[1]:])
        seen = [i for i in range(c.cu[1]) if i not in keep]
        assert bool(out[seen].isnan().any(-1).all())
    # a cached key that only the tokens nearest to the cache still see
    c = Case([100], [4], 8, 2, 128, 16, F16, window=40, mask=None, seed=12)
    clean, _ = c.check(D)
    c.vc[c.table[0, 62 // 16].long(), 62 % 16] = float("inf")  # position 62: seen from 100 and 101 only
    out, _ = c.call(D)
    assert torch.equal(out[2:], clean[2:]) and bool((~out[:2].isfinite()).all())


def test_tree_attention_through_an_overlapping_view(D):
    """Rings [slot, head, column, dim] of 64 + 1 columns read as pages of 16 rows, by a strided view and cyclic tables."""
    slots, hkv, cols, dim, window = 3, 2, 65, 128, 64
    g = torch.Generator(device="cuda").manual_seed(4)
    rk, rv = (torch.randn(slots, hkv, cols, dim, generator=g, device="cuda").half() for _ in range(2))
    lens, counts = [40, 64, 1000], [3, 1, 7]
    rows = slots * hkv * cols - (hkv - 1) * cols - 15
    view = [x.as_strided((rows, 16, hkv, dim), (dim, dim, cols * dim, 1)) for x in (rk, rv)]
    width = -(-max(lens) // 16)
    table = dev([[s * hkv * cols + 16 * (j % 4) for j in range(width)] for s in range(slots)])
    c = Case(lens, counts, 4, hkv, dim, 16, F16, window=window, seed=2)
    c.kc, c.vc, c.table = view[0], view[1], table
    c.check(D)


def test_tree_attention_offsets_beyond_32_bits(D):
    """Pages past element 2^31 of their pool."""
    page, hkv, dim = 64, 8, 128
    pages = (1 << 31) // (page * hkv * dim) + 40
    c = Case([1000, 70], [5, 3], 16, hkv, dim, page, F16, seed=9)
    kc, vc = (torch.empty(pages, page, hkv, dim, dtype=F16, device="cuda") for _ in range(2))
    n = c.kc.shape[0]
    kc[pages - n:], vc[pages - n:] = c.kc, c.vc
    c.kc, c.vc = kc, vc
    c.table = torch.where(c.table >= 0, c.table + pages - n, c.table)
    c.check(D)
    k, v = (torch.randn(4, hkv, dim, device="cuda").half() for _ in range(2))
    top = (pages - 1) * page
    D.store_rows(k, v, kc, vc, dev([top, top + 63, top + 5, top + 6]))
    assert torch.equal(kc[pages - 1][[0, 63, 5, 6]], k) and torch.equal(vc[pages - 1][[0, 63, 5, 6]], v)


def test_tree_attention_repeats_bit_for_bit_and_on_other_streams(D):
    c = Case([5000, 31, 900], [9, 4, 30], 32, 8, 128, 16, BF16, seed=21)
    out, lse = c.check(D)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    results = []
    with torch.cuda.stream(side):
        for _ in range(3):
            results.append(c.call(D))
    for _ in range(3):
        results.append(c.call(D))
    torch.cuda.synchronize()
    for o, s in results:
        assert torch.equal(o, out) and torch.equal(s, lse)


def test_tree_attention_in_a_graph(D):
    c = Case([700, 90], [5, 8], 8, 2, 256, 16, F16, window=512, seed=22)
    out, lse = c.check(D)
    lens, cu = dev(c.lens), dev(c.cu)
    ws = torch.empty(D.attention_workspace(256), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, s = D.tree_attention(c.q, c.k, c.v, c.kc, c.vc, c.table, lens, cu, c.scale, c.max_tree, c.mask, c.positions,
                                c.window, workspace=ws)
    for _ in range(2):
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, out) and torch.equal(s, lse)


def test_tree_attention_records_bad_indexes(D):
    err = err_word()
    c = Case([100, 50], [4, 4], 8, 2, 128, 16, F16, seed=1)
    good = c.table.clone()
    for value in (-1, c.kc.shape[0], 1 << 30):
        c.table = good.clone()
        c.table[1, 1] = value
        c.call(D, err=err)
        assert int(err.item()) == 6
        err.zero_()
    c.table = good
    lens = list(c.lens)
    for bad in (-1, 16 * good.shape[1] + 1):
        c.lens = [lens[0], bad]
        c.call(D, err=err)
        assert int(err.item()) == 5
        err.zero_()
    c.lens = lens
    c.cu = [0, 3, 7]
    c.max_tree = 3
    c.call(D, err=err)  # request 1 drafts four
    assert int(err.item()) == 5
    err.zero_()
    for cu in ([0, 4, 9], [0, -3, 8], [-1, 4, 8]):
        c.max_tree, c.cu = 16, cu
        c.call(D, err=err, mask=None)
        assert int(err.item()) == 5
        err.zero_()


# ---- store_rows -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("count,rows,heads,dim,page,dtype,heads_first,source", [
    (1, 1, 1, 64, 8, F16, False, False), (5, 40, 2, 256, 16, F16, True, True), (3000, 4000, 8, 128, 64, BF16, False, True),
    (77, 80, 3, 64, 24, BF16, True, False)])
def test_store_rows(D, count, rows, heads, dim, page, dtype, heads_first, source):
    g = torch.Generator(device="cuda").manual_seed(count)
    x = torch.randn(rows, 3, heads, dim, generator=g, device="cuda").to(dtype)
    k, v = x[:, 0], x[:, 2]
    pages = -(-count // page) + 2
    shape = (pages, heads, page, dim) if heads_first else (pages, page, heads, dim)
    kc, vc = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
    if heads_first:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    cg = torch.Generator().manual_seed(count)
    slots = torch.randperm(pages * page, generator=cg)[:count].tolist()
    src = torch.randint(0, rows, (count,), generator=cg).tolist() if source else list(range(count))
    if count > 10:
        slots[4] = -3
    want_k, want_v = kc.reshape(-1, heads, dim).cpu(), vc.reshape(-1, heads, dim).cpu()
    for s, i in zip(slots, src):
        if s >= 0:
            want_k[s], want_v[s] = k[i].cpu(), v[i].cpu()
    err = err_word()
    D.store_rows(k, v, kc, vc, dev(slots), dev(src) if source else None, err)
    assert int(err.item()) == 0
    assert torch.equal(kc.reshape(-1, heads, dim).cpu(), want_k) and torch.equal(vc.reshape(-1, heads, dim).cpu(), want_v)


def test_store_rows_records_bad_indexes(D):
    k = torch.ones(4, 2, 64, device="cuda").half()
    kc, vc = (torch.zeros(3, 8, 2, 64, device="cuda").half() for _ in range(2))
    for slots, source in (([24], [0]), ([0], [4]), ([0], [-1]), ([2 ** 31 - 1], [0])):
        err = err_word()
        D.store_rows(k, k, kc, vc, dev(slots), dev(source), err)
        assert int(err.item()) == 3
    assert not bool(kc.any())


# ---- refusals -------------------------------------------------------------------------------------------------------
def test_refusals(D):
    c = Case([40], [3], 8, 2, 128, 16, F16, seed=1)
    lens, cu = dev(c.lens), dev(c.cu)

    def attend(**kw):
        a = dict(q=c.q, k=c.k, v=c.v, k_cache=c.kc, v_cache=c.vc, table=c.table, lens=lens, cu=cu, scale=1.0, max_tree=3,
                 mask=c.mask, positions=c.positions)
        a.update(kw)
        return D.tree_attention(**a)

    attend()
    odd = torch.zeros(3, 8, 132, device="cuda", dtype=F16)
    bad = [dict(q=c.q.float()), dict(q=c.q.cpu()), dict(q=c.q[:, :7]), dict(k=c.k.bfloat16()), dict(k=c.k[:2]),
           dict(v=c.v[:, :1]), dict(q=odd[:, :, 1:129]), dict(k_cache=c.kc[:, :, :1]), dict(k_cache=c.kc[:, :9]),
           dict(v_cache=c.vc.transpose(1, 2).contiguous().transpose(1, 2)), dict(table=c.table.long()),
           dict(table=c.table[0]), dict(lens=lens[:0]), dict(lens=lens.long()), dict(cu=cu[:1]), dict(mask=c.mask.long()),
           dict(mask=c.mask[:2]), dict(max_tree=0), dict(max_tree=1025), dict(max_tree=33), dict(max_tree=3.0),
           dict(window=-1), dict(positions=c.positions[:1]), dict(positions=c.positions.float()),
           dict(err=torch.zeros(2, dtype=torch.int32, device="cuda")), dict(workspace=torch.zeros(4, device="cuda")),
           dict(k_cache=c.kc[:, :12], v_cache=c.vc[:, :12])]
    for kw in bad:
        with pytest.raises(ValueError):
            attend(**kw)
    for dim in (32, 96):
        with pytest.raises(ValueError):
            x = torch.zeros(3, 2, dim, device="cuda", dtype=F16)
            kc = torch.zeros(5, 16, 2, dim, device="cuda", dtype=F16)
            attend(q=x, k=x, v=x, k_cache=kc, v_cache=kc)
    w, inv = torch.ones(128, device="cuda"), torch.ones(32, device="cuda")
    pos = c.positions
    D.norm_rope(c.q, c.k, c.v, w, w, inv, pos, 1e-6, F16)
    for args in ((c.q, c.k, c.v, w[:64], w, inv, pos, 1e-6, F16), (c.q, c.k, c.v, w, w, inv, pos, 1e-6, F32),
                 (c.q, c.k, c.v, w, w, inv[:3], pos, 1e-6, F16), (c.q, c.k.float(), c.v, w, w, inv, pos, 1e-6, F16),
                 (c.q, c.k, c.v, w, w, torch.ones(72, device="cuda"), pos, 1e-6, F16),
                 (c.q, c.k, c.v, w, w, inv, pos.long(), 1e-6, F16), (c.q, c.k, c.v, w.half(), w, inv, pos, 1e-6, F16)):
        with pytest.raises(ValueError):
            D.norm_rope(*args)
    with pytest.raises(ValueError):
        D.norm_rope_store(c.q, c.k, c.v, w, w, inv, pos, 1e-6, c.kc.float(), c.vc.float(), pos)
    with pytest.raises(ValueError):
        D.store_rows(c.k, c.v, c.kc, c.vc, dev([0, 1, 2, 3]))
    with pytest.raises(ValueError):
        D.store_rows(c.k, c.v, c.kc.bfloat16(), c.vc.bfloat16(), dev([0]))
    for max_tree in (0, 2000, "3"):
        with pytest.raises(ValueError):
            D.plan_tree(dev([-1]), dev([0, 1]), dev([0]), max_tree)
    with pytest.raises(ValueError):
        D.plan_tree(dev([-1]), dev([0]), dev([0]), 1)
    ring, counters = dev([0, 1]), dev([0, 2], torch.int64)
    for a in ((dev([0]), dev([0, 1]), dev([[0]]), ring, counters, 16, 4), (dev([0]), dev([0]), dev([[0], [0]]), ring, counters, 16, 4),
              (dev([0]), dev([0]), dev([[0]]), ring, dev([0, 2]), 16, 4), (dev([0]), dev([0]), dev([[0]]), ring, counters, 0, 4),
              (dev([0]), dev([0]), dev([[0]]), ring, counters, 16, -1),
              (torch.zeros(4097, dtype=torch.int32, device="cuda"),) * 2 + (torch.zeros(4097, 1, dtype=torch.int32, device="cuda"), ring, counters, 16, 4)):
        with pytest.raises(ValueError):
            D.advance_tables(*a)


def test_empty_calls(D):
    c = Case([10, 20], [0, 0], 8, 2, 64, 16, F16, max_tree=4, mask=None)
    out, lse = c.call(D)
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8)
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    positions, mask = D.plan_tree(e, dev([0, 0, 0]), dev([10, 20]), 4)
    assert positions.shape == (0,) and mask.shape == (0, 1)
    D.store_rows(c.k, c.v, c.kc, c.vc, e)
    q, k, v = D.norm_rope(c.q, c.k, c.v, torch.ones(64, device="cuda"), torch.ones(64, device="cuda"),
                          torch.ones(32, device="cuda"), e, 1e-6, F16)
    assert q.shape == (0, 8, 64) and k.shape == (0, 2, 64)


# ---- the cache and the whole path -----------------------------------------------------------------------------------
def test_cache_grows_by_accepted_branches(D):
    """Two requests, three ticks: drafts attended, a branch accepted, its keys stored; the cache then holds exactly the
    accepted rows, and a finished request's pages serve another."""
    layers, hq, hkv, dim, page = 2, 4, 2, 64, 8
    cache = D.DraftCache(layers, rows=2, pages=6, page_size=page, max_len=40, kv_heads=hkv, dim=dim)
    g = torch.Generator(device="cuda").manual_seed(0)
    held = [[[], []], [[], []]]  # [layer][request]: accepted (k, v)
    for tick, (paths, n) in enumerate([(([0, 2], [1]), 4), (([0, 1, 3], []), 5), (([2], [0, 4]), 6)]):
        parents = dev([-1, -1, 0, 1, 0, 1][:n] * 2)
        parents[3] = 1
        cu = dev([0, n, 2 * n])
        positions, mask = D.plan_tree(parents, cu, cache.lens, n)
        kv = []
        for layer in range(layers):
            q = torch.randn(2 * n, hq, dim, generator=g, device="cuda").half()
            k, v = (torch.randn(2 * n, hkv, dim, generator=g, device="cuda").half() for _ in range(2))
            out, lse = cache.attend(layer, q, k, v, cu, 0.125, n, mask, positions)
            kv.append((k, v))
            c = Case([len(held[layer][b]) for b in range(2)], [n, n], hq, hkv, dim, page, F16, mask=None)
            c.q, c.k, c.v, c.kc, c.vc, c.table, c.mask = q, k, v, cache.k[layer], cache.v[layer], cache.table, mask
            c.bits = [int(x) for x in mask[:, 0].tolist()]
            c.positions = positions
            c.check(D)
        t = cache.advance(dev([len(p) for p in paths]), 8)
        flat = [i for p in ([paths[0]] + [[n + i for i in paths[1]]]) for i in p]
        source = dev(flat + [0] * (8 - len(flat)))
        for layer, (k, v) in enumerate(kv):
            cache.store(layer, k, v, t.slots, source)
            for b, p in enumerate(paths):
                held[layer][b] += [(k[b * n + i], v[b * n + i]) for i in p]
        cache.raise_device_error()
        assert cache.lens.tolist() == [len(held[0][b]) for b in range(2)]
    for layer in range(layers):
        for b in range(2):
            for i, (k, v) in enumerate(held[layer][b]):
                p = int(cache.table[b, i // page])
                assert torch.equal(cache.k[layer, p, i % page], k) and torch.equal(cache.v[layer, p, i % page], v)
    cache.advance(dev([-100, 0]), 0)
    cache.advance(dev([40, 0]), 40)  # five of six pages: the other request keeps its one
    assert cache.lens.tolist() == [40, 3] and cache.counters.tolist()[1] - cache.counters.tolist()[0] == 0
    cache.raise_device_error()
