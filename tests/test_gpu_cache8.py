"""The 8-bit cache (append_8bit, attention_8bit, DraftCache8) on a B200 against plain 64-bit implementations.

Scales, codes without a rotation and codes that a risen scale moves are equal bit by bit. Tolerances, u the result type's unit
roundoff (2^-11 fp16, 2^-8 bf16):
  codes after a rotation   half a step of e4m3: 2^-4 |y| or 2^-10 where y = x / scale is below the normal range, + 1e-5 of the
                           row's largest |y| for the fp32 arithmetic (two products and an angle, some roundings of 2^-24)
  q after a rotation       u |y| + 1e-5 of the row's largest |y|
  attention                u |o| for the result's rounding + (2^-11 + 2 ds + r) sum_j p_j |v_j|: 2^-11 for the weights, which
                           enter the second product in fp16 for both types, ds = dim 2^-23 scale max |q|.|k| for the fp32 sums of
                           the scores (a tensor core may cut where it adds), twice in a weight, r = (n / 8 + 32) 2^-23 for the sums
                           over n keys in 8 parts and their joining
  log-sum-exp              ds + r + 4e-6 (1 + |lse|)
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


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


def codes(x):
    """e4m3 codes of fp32 values as bytes, and NaN for what is not finite."""
    x = torch.where(x.abs() < math.inf, x, math.nan).cpu()
    return x.to(F8).view(torch.uint8)


def pool(pages, page, hkv, dim, heads_first=False, fill=None, seed=0):
    """[pages, page, hkv, dim] of random codes (none NaN), heads or tokens outermost within a page."""
    g = torch.Generator().manual_seed(seed)
    shape = (pages, hkv, page, dim) if heads_first else (pages, page, hkv, dim)
    x = codes(torch.randn(shape, generator=g) * 60) if fill is None else torch.full(shape, fill, dtype=torch.uint8)
    x = x.view(F8).cuda()
    return x.transpose(1, 2) if heads_first else x


# ---- append_8bit ----------------------------------------------------------------------------------------------------
def scale_for(bound):
    e = -100
    while e < 120 and bound > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def turned(x, positions, inv, pairs, factor):
    """Rows [n, heads, dim] in 64 bits with the first dims turned, and what each pair counts for the scale (fp32)."""
    rot = 2 * len(inv)
    angle = positions.double()[:, None, None] * inv.double()
    y = x.double().clone()
    size = x.float().abs().double()
    if rot:
        a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if pairs else (y[..., :rot // 2], y[..., rot // 2:rot])
        c, s = torch.cos(angle) * factor, torch.sin(angle) * factor
        p, q = a * c - b * s, b * c + a * s
        both = ((a.abs() + b.abs()).float() * torch.tensor(abs(factor), dtype=torch.float32)).double()
        y = torch.cat([torch.stack([p, q], -1).flatten(-2) if pairs else torch.cat([p, q], -1), y[..., rot:]], -1)
        size = torch.cat([both, both, size[..., rot:]], -1)
    return y, size


def append_reference(s, k, v, slots, source, positions, inv, pairs, factor):
    """Codes (bytes; values / scale in 64 bits for the new rows) and scales after the call, block by block."""
    page = s["kc"].shape[1]
    block = page // s["ks"].shape[1]
    out = {}
    rows = [i if source is None else source[i] for i in range(len(slots))]
    for name, x, rotate in (("k", k, True), ("v", v, False)):
        old = s[name + "c"].view(torch.uint8).cpu().clone()
        scale = s[name + "s"].cpu().clone()
        exact = torch.full(old.shape, math.nan, dtype=torch.float64)
        y, size = turned(x.cpu()[rows], positions, inv if rotate else inv[:0], pairs, factor)
        size = torch.where(size < math.inf, size, 0.0).amax(-1)
        written = {}
        for i, slot in enumerate(slots):
            if slot >= 0:
                written.setdefault(slot // block, []).append(i)
        for where, entries in written.items():
            pg, blk = where * block // page, where % (page // block)
            first = min(slots[i] % block for i in entries)
            for h in range(x.shape[1]):
                need = scale_for(max(float(size[i, h]) for i in entries))
                was = float(scale[pg, blk, h])
                new = need if first == 0 else max(need, was)
                if first and new > was:
                    at = slice(blk * block, blk * block + first)
                    moved = old[pg, at, h].view(F8).float() * (was / new)
                    old[pg, at, h] = codes(moved)
                scale[pg, blk, h] = new
                for i in entries:
                    exact[pg, slots[i] % page, h] = y[i, h] / new
        out[name] = old, exact, scale
    return out


def check_append(s, ref, rotated):
    for name in ("k", "v"):
        old, exact, scale = ref[name]
        assert torch.equal(s[name + "s"].cpu(), scale), name
        got = s[name + "c"].cpu()
        fresh = ~torch.isnan(exact)
        if rotated and name == "k":
            assert torch.equal(got.view(torch.uint8)[~fresh], old[~fresh])
            y, g = exact[fresh], got.float().double()[fresh]
            most = torch.where(fresh, exact.abs(), 0.0).amax(-1, keepdim=True).expand_as(exact)[fresh]
            assert bool(((g - y).abs() <= torch.clamp(2.0 ** -4 * y.abs(), min=2.0 ** -10) + 1e-5 * most).all())
        else:
            want = torch.where(fresh, codes(exact.float()), old)
            assert torch.equal(got.view(torch.uint8), want), name


def append_state(pages, page, block, hkv, dim, heads_first, seed):
    g = torch.Generator().manual_seed(seed)
    s = {"kc": pool(pages, page, hkv, dim, heads_first, seed=seed), "vc": pool(pages, page, hkv, dim, heads_first, seed=seed + 1)}
    for name in ("ks", "vs"):
        s[name] = torch.exp2(torch.randint(-9, -3, (pages, page // block, hkv), generator=g).float()).cuda()
    return s


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,hq,hkv,rot,pairs,factor,page,block,heads_first,counts", [
    (64, 0, 1, 0, False, 1.0, 8, 8, False, [1]),
    (64, 7, 1, 64, True, 1.0, 24, 8, True, [1, 0, 3, 30]),
    (128, 8, 8, 32, False, 0.8, 16, 16, False, [5, 16, 17, 1]),
    (128, 32, 8, 128, True, 1.2079, 64, 32, True, [100, 1, 33]),
    (256, 8, 2, 64, False, 1.0, 16, 8, False, [40, 2, 2, 1, 1, 9]),
    (256, 2, 2, 256, False, -1.5, 128, 128, True, [200, 3]),
    (128, 4, 4, 16, True, 1.0, 48, 24, False, [1] * 40),
])
def test_append(D, dim, hq, hkv, rot, pairs, factor, page, block, heads_first, counts, dtype):
    g = torch.Generator().manual_seed(dim + rot + page)
    starts = [int(x) for x in torch.randint(0, 2 * page, (len(counts),), generator=g)]
    starts[0] = 0
    slots, positions, at = [], [], 0
    for n, a in zip(counts, starts):
        held = -(-(a + n) // page)
        order = [at + (3 * j + 1) % held if held % 3 else at + j for j in range(held)]
        slots += [order[(a + i) // page] * page + (a + i) % page for i in range(n)]
        positions += [a + i + 70000 * (n % 2) for i in range(n)]
        at += held
    if len(slots) > 4:
        slots[2] = -1
    total = len(slots)
    s = append_state(at + 1, page, block, hkv, dim, heads_first, 5)
    width = hq + 2 * hkv
    x = (torch.randn(total, width * dim, generator=g) * torch.exp2(torch.randint(-6, 4, (total, 1), generator=g).float())).to(dtype).cuda()
    q, k, v = (x[:, a * dim:b * dim].view(total, b - a, dim) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, width)))
    inv = 10000.0 ** (-torch.arange(0, rot, 2).float() / max(1, rot))
    p = torch.tensor(positions, dtype=torch.int32)
    ref = append_reference(s, k, v, slots, None, p, inv, pairs, factor)
    err = err_word()
    for _ in range(2):  # the same call again changes nothing
        got = D.append_8bit(k, v, s["kc"], s["vc"], s["ks"], s["vs"], dev(slots), positions=p.cuda() if rot else None,
                            inv_freq=inv.cuda() if rot else None, interleaved=pairs, rope_scale=factor, q=q if hq else None, err=err)
        assert int(err.item()) == 0
        check_append(s, ref, rot > 0)
        if hq:
            y, _ = turned(q.cpu(), p, inv, pairs, factor)
            assert got.dtype == dtype and got.is_contiguous()
            assert bool(((got.cpu().double() - y).abs() <= U[dtype] * y.abs() + 1e-5 * y.abs().amax(-1, keepdim=True) + 2.0 ** -25).all())
        else:
            assert got is None


def test_append_source_and_many_entries(D):
    """Rows picked by a source, more entries than one a thread block."""
    g = torch.Generator().manual_seed(3)
    pages, page, hkv, dim = 700, 16, 2, 64
    s = append_state(pages, page, 8, hkv, dim, False, 6)
    n = 5000
    rows = torch.randperm(6000, generator=g)[:n]
    k, v = (torch.randn(6000, hkv, dim, generator=g).to(F16).cuda() for _ in range(2))
    order = torch.randperm(pages, generator=g)
    slots = (order[torch.arange(n) // page] * page + torch.arange(n) % page).tolist()
    ref = append_reference(s, k, v, slots, rows.tolist(), torch.zeros(n), torch.zeros(0), False, 1.0)
    D.append_8bit(k, v, s["kc"], s["vc"], s["ks"], s["vs"], dev(slots), source=rows.int().cuda())
    check_append(s, ref, False)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_values_at_the_edge(D, dtype):
    """Zeros, the smallest and the largest numbers, a border between two scales, infinities and NaN (which spare the others)."""
    page, hkv, dim = 16, 1, 64
    s = append_state(12, page, 16, hkv, dim, False, 7)
    top = torch.finfo(dtype).max
    k = torch.zeros(12, hkv, dim)
    k[1, 0, 5] = torch.finfo(dtype).smallest_normal
    k[2, 0, 5], k[2, 0, 6] = top, -top / 3
    k[3, 0, 7] = 448.0 * 2.0 ** -3
    k[4, 0, 7] = 449.0 * 2.0 ** -3 if dtype == F16 else 450.0 * 2.0 ** -3
    k[5] = 1.0
    k[5, 0, 1], k[5, 0, 2], k[5, 0, 3] = math.inf, -math.inf, math.nan
    k[6] = math.nan
    k[7:] = torch.randn(5, 1, dim)
    k = k.to(dtype).cuda()
    slots = [16 * i + 0 for i in range(12)]
    ref = append_reference(s, k, k, slots, None, torch.zeros(12), torch.zeros(0), False, 1.0)
    D.append_8bit(k, k, s["kc"], s["vc"], s["ks"], s["vs"], dev(slots))
    got, raw = s["kc"].float().cpu(), s["kc"].view(torch.uint8).cpu()
    for name in ("k", "v"):
        assert torch.equal(s[name + "s"].cpu(), ref[name][2])
    assert torch.isnan(got[5, 0, 0, 1:4]).all() and torch.isnan(got[6, 0]).all()
    assert float(s["ks"][5, 0, 0]) == 2.0 ** -8 and bool((got[5, 0, 0, 4:] == 256).all())
    want = codes((k.float().cpu() / ref["k"][2][:, 0, :, None])[:, 0])
    assert torch.equal(raw[:, 0, 0][torch.isfinite(k.cpu().float()[:, 0])], want[torch.isfinite(k.cpu().float()[:, 0])])
    assert float(s["ks"][0, 0, 0]) == 2.0 ** -100 and bool((raw[0, 0] == 0).all())


def test_append_a_scale_that_rises_and_one_that_stays(D):
    page, dim = 32, 128
    s = append_state(2, page, 16, 2, dim, True, 8)
    for step, (first, n, size) in enumerate([(0, 3, 1.0), (3, 5, 0.01), (8, 1, 30.0), (9, 1, 1e-6), (10, 12, 500.0), (22, 1, 1.0)]):
        g = torch.Generator().manual_seed(step)
        k, v = ((torch.randn(n, 2, dim, generator=g) * size).to(BF16).cuda() for _ in range(2))
        slots = list(range(page + first, page + first + n))
        ref = append_reference(s, k, v, slots, None, torch.zeros(n), torch.zeros(0), False, 1.0)
        D.append_8bit(k, v, s["kc"], s["vc"], s["ks"], s["vs"], dev(slots))
        check_append(s, ref, False)


@pytest.mark.parametrize("pad", [1, 31, 33, 200])
def test_append_of_a_padded_batch(D, pad):
    """Entries that are skipped before, within and after a block's: queries of all of them are turned, the block is one."""
    page, hkv, hq, dim = 64, 2, 6, 128
    s = append_state(5, page, 32, hkv, dim, False, 20)
    slots = [-1] * pad + [64, 65] + [-1] * pad + [66, 67, 96] + [-1] * pad + [130] + [-1] * pad + [131] * 1 + [-1] * pad
    n = len(slots)
    g = torch.Generator().manual_seed(pad)
    x = torch.randn(n, hq + 2 * hkv, dim, generator=g).bfloat16().cuda()
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    inv = 10000.0 ** (-torch.arange(0, 64, 2).float() / 64)
    p = torch.arange(n, dtype=torch.int32) * 7
    ref = append_reference(s, k, v, slots, None, p, inv, False, 1.0)
    err = err_word()
    got = D.append_8bit(k, v, s["kc"], s["vc"], s["ks"], s["vs"], dev(slots), positions=p.cuda(), inv_freq=inv.cuda(), q=q, err=err)
    assert int(err.item()) == 0
    check_append(s, ref, True)
    y, _ = turned(q.cpu(), p, inv, False, 1.0)
    assert bool(((got.cpu().double() - y).abs() <= U[BF16] * y.abs() + 1e-5 * y.abs().amax(-1, keepdim=True)).all())


def test_append_far_positions(D):
    """Angles of positions up to 2^31 - 1, and of negative ones, to fp32's own exactness."""
    page, dim = 16, 64
    s = append_state(2, page, 16, 1, dim, False, 21)
    p = torch.tensor([0, 1, 65537, 1 << 24, (1 << 24) + 1, 1 << 30, 2 ** 31 - 1, -5], dtype=torch.int32)
    inv = torch.cat([torch.tensor([1.0, 0.9999999, 3.1, 7.5, 100.25]), 500000.0 ** (-torch.arange(0, 54, 2).float() / 64)])
    x = torch.randn(8, 3, dim, generator=torch.Generator().manual_seed(2)).half().cuda()
    q = D.append_8bit(x[:, :1], x[:, 1:2], s["kc"], s["vc"], s["ks"], s["vs"], dev(range(8)), positions=p.cuda(), inv_freq=inv.cuda(), q=x[:, 2:])
    y, _ = turned(x[:, 2:].cpu(), p, inv, False, 1.0)
    # 2^31 positions times 2^-53 of a frequency of up to 100 / (2 pi) turns: below 2^-18 of a turn there, 1e-6 at ordinary ones
    angle = p.double().abs()[:, None, None] * inv.double().abs() * 2.0 ** -52
    slack = 1e-6 + torch.cat([angle, angle], -1)
    assert bool(((q.cpu().double() - y).abs() <= U[F16] * y.abs() + slack * 8 + 1e-6).all())


def test_append_refuses_slots_on_the_device(D):
    """Slots beyond the pages, ones that do not ascend in a block, sources outside the rows: recorded, the rest is written."""
    page, hkv, dim = 16, 2, 64
    k = torch.randn(6, hkv, dim, device="cuda").half()
    for slots, source, good in (([0, 1, 4 * 16, 17, -1, 33], None, [0, 1, 3, 5]), ([0, 1, 1, 16, 17, 18], None, [0, 1, 3, 4, 5]),
                                ([5, 4, 16, 17, 32, 33], None, [0, 2, 3, 4, 5]), ([0, 1, 2, 16, 17, 18], [0, 1, 2, 3, 6, -1], [0, 1, 2, 3])):
        s = append_state(4, page, 16, hkv, dim, False, 9)
        before = {n: x.view(torch.uint8).cpu().clone() if x.dtype == F8 else x.cpu().clone() for n, x in s.items()}
        kept = [x if i in good else -1 for i, x in enumerate(slots)]
        ref = append_reference(s, k, k, kept, [x if 0 <= x < 6 else 0 for x in source] if source else None, torch.zeros(6), torch.zeros(0), False, 1.0)
        err = err_word()
        D.append_8bit(k, k, s["kc"], s["vc"], s["ks"], s["vs"], dev(slots), source=dev(source) if source else None, err=err)
        assert int(err.item()) == 3
        check_append(s, ref, False)
        assert before["kc"].shape == s["kc"].shape


def test_append_nothing(D):
    s = append_state(2, 16, 8, 2, 64, False, 10)
    before = s["kc"].view(torch.uint8).clone()
    k = torch.zeros(0, 2, 64, dtype=F16, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert D.append_8bit(k, k, s["kc"], s["vc"], s["ks"], s["vs"], none) is None
    q = D.append_8bit(k, k, s["kc"], s["vc"], s["ks"], s["vs"], none, positions=none, inv_freq=torch.ones(16, device="cuda"), q=k)
    assert q.shape == (0, 2, 64) and torch.equal(before, s["kc"].view(torch.uint8))


# ---- attention_8bit -------------------------------------------------------------------------------------------------
def attention_state(dim, hq, hkv, page, block, lens, counts, dtype, heads_first=False, tree=False, spread=(-8, -5), seed=0, pad=0):
    g = torch.Generator().manual_seed(seed)
    rows, total = len(lens), sum(counts)
    held = [-(-n // page) for n in lens]
    pages = sum(held) + 2
    order = torch.randperm(pages, generator=g).tolist()
    width = max(1, max(held)) + pad
    table, at = [], 0
    for h in held:
        table.append(order[at:at + h] + [-7] * (width - h))
        at += h
    s = {"kc": pool(pages, page, hkv, dim, heads_first, seed=seed + 1), "vc": pool(pages, page, hkv, dim, heads_first, seed=seed + 2)}
    for name in ("ks", "vs"):
        s[name] = torch.exp2(torch.empty(pages, page // block, hkv).uniform_(*spread, generator=g)).cuda()
    # what no token has filled: NaN codes, NaN scales
    for name in ("k", "v"):
        raw = s[name + "c"].view(torch.uint8)
        for p in order[at:]:
            raw[p] = 0x7f
            s[name + "s"][p] = math.nan
        for b, n in enumerate(lens):
            if n % page:
                raw[table[b][n // page], n % page:] = 0xff
                first = -(-(n % page) // block)
                s[name + "s"][table[b][n // page], first:] = math.nan
    wide = torch.randn(total, hq + 2, dim, generator=g).to(dtype).cuda()
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    s.update(q=wide[:, 1:1 + hq], table=dev(table), lens=dev(lens), cu=dev(cu), mask=None, positions=None)
    if tree:
        words = max(1, -(-max(counts) // 32))
        bits = torch.zeros(total, words * 32, dtype=torch.bool)
        pos = []
        for b, c in enumerate(counts):
            for t in range(c):
                parent = -1 if t == 0 else int(torch.randint(-1, t, (1,), generator=g))
                if parent >= 0:
                    bits[cu[b] + t] = bits[cu[b] + parent]
                bits[cu[b] + t, t] = True
                pos.append(lens[b] - c + int(bits[cu[b] + t].sum()) - 1)
        packed = (bits.view(total, words, 32).long() * (1 << torch.arange(32))).sum(-1)
        s["mask"] = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).int().cuda()
        s["positions"] = dev(pos)
    return s


def attention_reference(s, scale, window=0, sinks=0, use_positions=True):
    """Token by token group: out, log-sum-exp, tolerance of both (before the result's rounding)."""
    q, lens, cu = s["q"], s["lens"].tolist(), s["cu"].tolist()
    page, hkv, dim = s["kc"].shape[1:]
    block, group = page // s["ks"].shape[1], q.shape[1] // s["kc"].shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    for b, n in enumerate(lens):
        a, z = cu[b], cu[b + 1]
        if z == a:
            continue
        old = n - (z - a)
        j = torch.arange(n, device="cuda")
        where = s["table"][b].long()[j // page]
        t = torch.arange(z - a, device="cuda")
        pos = s["positions"][a:z].long() if s["positions"] is not None and use_positions else old + t
        kpos = torch.cat([j[:old], pos]) if s["positions"] is not None and use_positions else j
        if s["mask"] is None:
            new = t <= t[:, None]
        else:
            m = s["mask"][a:z].long() & 0xffffffff
            new = (m[:, t // 32] >> (t % 32)) & 1 != 0
        see = torch.cat([torch.ones(z - a, old, dtype=torch.bool, device="cuda"), new], 1)
        if window:
            see = see & ((kpos > pos[:, None] - window) | (kpos < sinks))
        for h in range(hkv):
            ks, vs = (s[x][where, j % page // block, h].double() for x in ("ks", "vs"))
            k, v = s["kc"][where, j % page, h].double() * ks[:, None], s["vc"][where, j % page, h].double() * vs[:, None]
            for r in range(z - a):  # a row sees exactly its own keys
                at = see[r].nonzero()[:, 0]
                if not len(at):
                    continue
                x = q[a + r, h * group:(h + 1) * group].double()
                score = x @ k[at].T * scale
                ds = dim * 2.0 ** -23 * scale * (x.abs() @ k[at].abs().T).amax(-1)
                whole = torch.logsumexp(score, -1)
                p = torch.exp(score - whole[:, None])
                p = torch.where(torch.isneginf(whole)[:, None], 0.0, p)
                heads = slice(h * group, (h + 1) * group)
                out[a + r, heads] = p @ v[at]
                lse[a + r, heads] = whole
                more = (len(at) / 8 + 32) * 2.0 ** -23
                tol[a + r, heads] = (2.0 ** -11 + 2 * ds + more)[:, None] * (p @ v[at].abs())
                ltol[a + r, heads] = ds + more + 4e-6 * (1 + whole.abs())
    return out, lse, tol, ltol


def check_attention(got, ref, dtype):
    (out, lse), (o, l, tol, ltol) = got, ref
    assert out.dtype == dtype and lse.dtype == torch.float32
    # what is beyond the type's numbers becomes infinite; what may be on either side of their end is either
    limit = torch.finfo(dtype).max
    over, near_end = o.abs() - tol > limit * (1 + U[dtype]), o.abs() * (1 + U[dtype]) + tol >= limit
    assert torch.equal(out.double()[over], torch.sign(o[over]) * math.inf)
    d = torch.where(near_end, 0.0, (out.double() - o).abs())
    assert bool((d <= U[dtype] * o.abs() + tol + 2.0 ** -25).all()), float((d / (U[dtype] * o.abs() + tol + 1e-30)).max())
    none = torch.isneginf(l)
    assert torch.equal(none, torch.isneginf(lse)) and bool((out[none] == 0).all())
    assert bool(((lse.double() - l).abs()[~none] <= ltol[~none]).all())


def attend(D, s, scale, max_new, **kw):
    return D.attention_8bit(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["lens"], s["cu"], scale, max_new,
                            mask=s["mask"], positions=s["positions"], **kw)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,hq,hkv,page,block,heads_first,lens,counts,window,sinks,tree", [
    (64, 1, 1, 8, 8, False, [1], [1], 0, 0, False),
    (64, 4, 4, 8, 8, True, [7, 8, 9, 128, 129, 3], [1, 1, 2, 1, 3, 3], 0, 0, False),
    (128, 8, 2, 16, 16, False, [100, 1, 0, 517, 40], [1, 1, 0, 2, 0], 0, 0, False),
    (128, 5, 5, 24, 8, False, [700, 65, 300], [5, 65, 1], 64, 3, False),
    (128, 32, 2, 64, 32, True, [1030, 130], [3, 1], 512, 4, False),
    (256, 8, 2, 16, 16, False, [2000, 513, 516, 20, 600], [1, 1, 2, 20, 1], 512, 4, False),
    (256, 6, 2, 48, 24, True, [333, 50], [33, 50], 0, 0, False),
    (256, 8, 2, 16, 8, False, [333, 50, 300], [33, 50, 7], 0, 0, True),
    (128, 32, 4, 32, 8, False, [400, 90, 64], [40, 3, 64], 0, 0, True),
    (64, 15, 5, 128, 128, True, [900, 33, 70], [33, 33, 70], 20, 0, True),
    (64, 7, 1, 16, 16, False, [900, 133, 70], [33, 33, 70], 200, 150, True),
    (128, 128, 1, 16, 16, False, [300], [4], 0, 0, False),
    (128, 16, 1, 64, 64, False, [20000], [1], 0, 0, False),
    (64, 2, 1, 8, 8, False, [9000, 3, 5000], [2, 1, 1], 1, 1, False),
])
def test_attention(D, dim, hq, hkv, page, block, heads_first, lens, counts, window, sinks, tree, dtype):
    s = attention_state(dim, hq, hkv, page, block, lens, counts, dtype, heads_first, tree, seed=dim + page, pad=2)
    err = err_word()
    got = attend(D, s, dim ** -0.5, max(counts), window=window, sinks=sinks, err=err)
    assert int(err.item()) == 0
    check_attention(got, attention_reference(s, dim ** -0.5, window, sinks), dtype)
    again = attend(D, s, dim ** -0.5, max(counts) + 5 if not tree else max(counts), window=window, sinks=sinks)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("dim,hq,hkv,n", [(128, 32, 4, 300), (64, 8, 8, 200), (256, 8, 2, 150), (128, 20, 1, 129)])
def test_attention_many_rows(D, dim, hq, hkv, n):
    """Chunks of prompts: more rows a key head than any tile has."""
    for dtype, window, sinks in ((F16, 0, 0), (BF16, 100, 5)):
        s = attention_state(dim, hq, hkv, 32, 16, [n, n + 411, 3, n + 40], [n, n // 2, 2, n], dtype, seed=n)
        got = attend(D, s, dim ** -0.5, n, window=window, sinks=sinks)
        check_attention(got, attention_reference(s, dim ** -0.5, window, sinks), dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n", [1, 40])
def test_attention_scales_far_apart(D, dtype, n):
    """V scales over 2^40: a row that only looks at small ones is as exact as any. K scales that make sharp rows."""
    s = attention_state(128, 8, 2, 16, 8, [500, 260], [n, n], dtype, spread=(-25, 15), seed=4)
    s["ks"] = torch.exp2(torch.empty(s["ks"].shape).uniform_(-9, -3, generator=torch.Generator().manual_seed(1))).cuda()
    # what lies beyond the lengths stays NaN
    got = attend(D, s, 0.3, n)
    check_attention(got, attention_reference(s, 0.3), dtype)


@pytest.mark.parametrize("n", [3, 50])
def test_attention_nan_is_for_those_who_see_it(D, n):
    """A NaN key or value among the new tokens or at a window's edge reaches the rows that see it and no other."""
    for tree, window, sinks in ((False, 0, 0), (True, 0, 0), (False, 90, 2)):
        s = attention_state(128, 8, 2, 16, 16, [200, 150], [n, n], F16, tree=tree, seed=11)
        clean = attend(D, s, 0.1, n, window=window, sinks=sinks)
        page = 16
        places = [(0, 200 - n + 1), (0, 200 - n - 91 + 3), (1, 150 - 1)]
        for b, j in places:
            p = int(s["table"][b, j // page])
            s["vc"].view(torch.uint8)[p, j % page, 1, 5] = 0x7f
            s["kc"].view(torch.uint8)[p, j % page, 0, 9] = 0xff
        got, lse = attend(D, s, 0.1, n, window=window, sinks=sinks)
        cu, lens = s["cu"].tolist(), s["lens"].tolist()
        bits = s["mask"].cpu().long() & 0xffffffff if tree else None
        for b in range(2):
            old = lens[b] - n
            for t in range(n):
                def sees(j):
                    if j >= old:
                        u = j - old
                        ok = u <= t if not tree else bool(bits[cu[b] + t, u // 32] >> (u % 32) & 1)
                    else:
                        ok = True
                    pos = old + t if not tree else int(s["positions"][cu[b] + t])
                    return ok and (not window or j > pos - window or j < sinks)
                hit = any(sees(j) for bb, j in places if bb == b)
                row = got[cu[b] + t]
                assert bool(torch.isnan(row[:4]).all()) == hit and bool(torch.isnan(row[:4]).any()) == hit, (tree, window, b, t)
                assert bool(torch.isnan(lse[cu[b] + t, :4]).all()) == hit
                assert bool(torch.isnan(row[4:, 5]).all()) == hit and not bool(torch.isnan(row[4:, :5]).any())
                assert not bool(torch.isnan(row[4:, 6:]).any())
                if not hit:
                    assert torch.equal(row, clean[0][cu[b] + t])


def test_attention_rows_that_see_nothing(D):
    """Masks without a bit over an empty cache, queries of infinities and NaN, scores of -inf."""
    s = attention_state(64, 4, 2, 16, 16, [5, 40], [5, 5], F16, tree=True, seed=12)
    s["mask"][2] = 0
    s["mask"][7] = 0
    q = s["q"].clone()
    q[1, 1] = math.nan
    s["q"] = q
    out, lse = attend(D, s, 0.125, 5)
    assert bool((out[2] == 0).all()) and bool(torch.isneginf(lse[2]).all())
    assert bool(torch.isnan(out[1, 1]).all()) and bool(torch.isnan(lse[1, 1])) and not bool(torch.isnan(out[1, [0, 2, 3]]).any())
    ref = attention_reference(s, 0.125)
    keep = torch.ones(10, 4, dtype=torch.bool, device="cuda")
    keep[1, 1] = False
    assert bool(((out.double() - ref[0]).abs()[keep] <= (U[F16] * ref[0].abs() + ref[2] + 2.0 ** -25)[keep]).all())


def test_attention_no_request_and_bad_lengths(D):
    """Tokens of no request, and of requests whose lengths are out of range, are 0 and -inf; the others are as they were."""
    s = attention_state(64, 4, 2, 16, 16, [50, 60, 70, 9], [2, 3, 1, 2], F16, seed=13)
    good = attend(D, s, 0.125, 3)
    cu = s["cu"].clone()
    wide = torch.cat([torch.full((4, 4, 64), math.nan, device="cuda").half(), s["q"], torch.full((9, 4, 64), math.nan, device="cuda").half()])
    lens = s["lens"].clone()
    lens[1], lens[3] = 16 * s["table"].shape[1] + 1, 1
    err = err_word()
    out, lse = D.attention_8bit(wide, s["kc"], s["vc"], s["ks"], s["vs"], s["table"], lens, cu + 4, 0.125, 3, err=err)
    assert int(err.item()) == 5
    blank = [0, 1, 2, 3] + [4 + 2, 4 + 3, 4 + 4] + [4 + 6, 4 + 7] + list(range(12, 21))
    assert bool((out[blank] == 0).all()) and bool(torch.isneginf(lse[blank]).all())
    # where a request's keys are cut, and so the order of its sums, goes by all requests of a call
    ref = attention_reference(s, 0.125)
    keep = [0, 1, 5]
    check_attention((out[4:][keep], lse[4:][keep]), [x[keep] for x in ref], F16)
    check_attention(good, ref, F16)
    out, lse = D.attention_8bit(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["lens"], s["cu"], 0.125, 2, err=err.zero_())
    assert int(err.item()) == 5 and bool((out[2:5] == 0).all())
    check_attention((out[:2], lse[:2]), [x[:2] for x in ref], F16)
    out, lse = D.attention_8bit(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"][:0], s["lens"][:0], s["cu"][:1], 0.125, 2)
    assert bool((out == 0).all()) and bool(torch.isneginf(lse).all())


def test_attention_records_a_bad_page(D):
    for bad in (-1, 1 << 20):
        s = attention_state(64, 4, 2, 16, 16, [50, 60], [1, 1], F16, seed=14)
        good = attend(D, s, 0.125, 1)
        s["table"][0, 1] = bad
        err = err_word()
        out, lse = attend(D, s, 0.125, 1, err=err)
        assert int(err.item()) == 6 and torch.equal(out[1], good[0][1])
        # pages that the window has left are not looked at
        err.zero_()
        attend(D, s, 0.125, 1, window=18, sinks=2, err=err)
        assert int(err.item()) == 0


def test_attention_many_requests(D):
    """More items than thread blocks, of all lengths, in one line."""
    g = torch.Generator().manual_seed(15)
    lens = [int(x) for x in torch.randint(0, 400, (300,), generator=g)]
    lens[7], lens[130] = 6000, 3000
    counts = [min(n, int(x)) for n, x in zip(lens, torch.randint(0, 3, (300,), generator=g))]
    for window, sinks in ((0, 0), (100, 4)):
        s = attention_state(64, 4, 2, 16, 16, lens, counts, BF16, seed=16)
        check_attention(attend(D, s, 0.125, 2, window=window, sinks=sinks), attention_reference(s, 0.125, window, sinks), BF16)


def test_attention_streams_and_graphs(D):
    """A call on a side stream, two at once, and a captured one replayed after its inputs changed."""
    s = attention_state(128, 8, 2, 16, 16, [700, 90], [2, 2], F16, seed=17)
    want = attend(D, s, 0.1, 2)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for st in streams:
        with torch.cuda.stream(st):
            for _ in range(20):
                o = attend(D, s, 0.1, 2)
            outs.append(o)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
    ws = torch.empty(D.attention_8bit_workspace(128, 4, 8), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = attend(D, s, 0.1, 2, workspace=ws)
    s["lens"].copy_(dev([650, 33]))
    s2 = dict(s)
    graph.replay()
    torch.cuda.synchronize()
    now = attend(D, s2, 0.1, 2)
    assert torch.equal(o[0], now[0]) and torch.equal(o[1], now[1]) and not torch.equal(o[0], want[0])


def test_attention_offsets_beyond_32_bits(D):
    """A pool of more than 2^32 bytes: pages at its far end."""
    dim, hkv, page = 256, 8, 128
    pages = (1 << 32) // (page * hkv * dim) + 40
    k, v = (torch.zeros(pages, page, hkv, dim, dtype=torch.uint8, device="cuda").view(F8) for _ in range(2))
    small = attention_state(dim, 16, hkv, page, 16, [300, 129], [1, 1], BF16, seed=18)
    n = small["kc"].shape[0]
    k.view(torch.uint8)[pages - n:] = small["kc"].view(torch.uint8)
    v.view(torch.uint8)[pages - n:] = small["vc"].view(torch.uint8)
    ks, vs = (torch.ones(pages, page // 16, hkv, device="cuda") for _ in range(2))
    ks[pages - n:], vs[pages - n:] = small["ks"], small["vs"]
    want = attend(D, small, 0.06, 1)
    table = torch.where(small["table"] >= 0, small["table"] + pages - n, -1).int()
    got = D.attention_8bit(small["q"], k, v, ks, vs, table, small["lens"], small["cu"], 0.06, 1)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    x = torch.randn(2, hkv, dim, device="cuda").half()
    slots = dev([(pages - 1) * page + 16, (pages - 1) * page + 17])
    D.append_8bit(x, x, k, v, ks, vs, slots)
    scale = ks[pages - 1, 1][:, None]
    assert bool(((k[pages - 1, 16:18].float() * scale - x.float()).abs() <= torch.clamp(x.float().abs() / 16, min=2.0 ** -10) * 1.001).all())


# ---- together -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("block,window,sinks", [(8, 0, 0), (16, 48, 4)])
def test_generation_over_draft_cache8(D, block, window, sinks):
    """Prompts in chunks, then tokens, some of them taken back: what attention gives is what the rows that were kept say, to the
    8 bits that they are kept in."""
    hq, hkv, dim, page, rows, scale = 8, 2, 64, 16, 3, 0.125
    cache = D.DraftCache8(2, rows, 60, page, 400, hkv, dim, block)
    assert cache.k.dtype == F8 and cache.k_scale.shape == (2, 60, page // block, hkv)
    inv = (10000.0 ** (-torch.arange(0, dim, 2).float() / dim)).cuda()
    g = torch.Generator().manual_seed(1)
    kept = [[] for _ in range(rows)]  # (turned k, v) rows in 64 bits
    for step, delta in enumerate([[70, 5, 0], [33, 1, 129], [1, 1, 1], [6, 4, 5], [-4, -1, -5], [1, 1, 1], [-80, 2, 1], [2, 1, 1]]):
        t = cache.advance(dev(delta), sum(max(0, d) for d in delta))
        new = [max(0, d) for d in delta]
        for b, d in enumerate(delta):
            if d < 0:
                del kept[b][d:]
        n = sum(new)
        if not n:
            continue
        x = torch.randn(n, hq + 2 * hkv, dim, generator=g).half().cuda()
        q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        layer = step % 2
        for other in (1 - layer, layer):  # both layers hold the same tokens
            rq = cache.store(other, k, v, t.slots, positions=t.positions, inv_freq=inv, interleaved=True, q=q)
        ky, _ = turned(k.cpu(), t.positions.cpu(), inv.cpu(), True, 1.0)
        i = 0
        for b, c in enumerate(new):
            for _ in range(c):
                kept[b].append((ky[i], v[i].cpu().double()))
                i += 1
        out, lse = cache.attend(layer, rq, t.cu, scale, max(new), window=window, sinks=sinks)
        i = 0
        for b, c in enumerate(new):
            if not c:
                continue
            K, V = (torch.stack([x[j] for x in kept[b]]) for j in (0, 1))
            for r in range(c):
                pos = len(kept[b]) - c + r
                j = torch.arange(pos + 1)
                if window:
                    j = j[(j > pos - window) | (j < sinks)]
                heads = rq[i].cpu().double().unflatten(0, (hkv, -1))
                score = torch.einsum("hgd,nhd->hgn", heads, K[j]) * scale
                # 8 bits: 2^-4 of each element, or what a scale that rose has left; three standard deviations of a sum
                p = torch.softmax(score, -1)
                ref = torch.einsum("hgn,nhd->hgd", p, V[j]).flatten(0, 1)
                noise = 2.0 ** -4 * scale * (heads.pow(2).sum(-1, keepdim=True) * 2.0).sqrt() + 2.0 ** -4
                far = (out[i].cpu().double() - ref).abs()
                assert float((far / (3 * noise.flatten(0, 1) * torch.einsum("hgn,nhd->hgd", p, V[j].abs()).flatten(0, 1) + 0.02)).max()) < 1
                i += 1
        assert torch.equal(cache.k[0].view(torch.uint8), cache.k[1].view(torch.uint8))
    cache.raise_device_error()


def test_refusals(D):
    s = attention_state(64, 4, 2, 16, 16, [50], [1], F16, seed=19)
    k = torch.zeros(1, 2, 64, device="cuda").half()
    slots = dev([3])

    def append(**kw):
        a = dict(k=k, v=k, k_cache=s["kc"], v_cache=s["vc"], k_scale=s["ks"], v_scale=s["vs"], slots=slots)
        a.update(kw)
        return D.append_8bit(**a)

    def attention(**kw):
        a = dict(q=s["q"], k_cache=s["kc"], v_cache=s["vc"], k_scale=s["ks"], v_scale=s["vs"], table=s["table"], lens=s["lens"],
                 cu=s["cu"], scale=0.1, max_new=1)
        a.update(kw)
        return D.attention_8bit(**a)

    append()
    attention()
    half, one = torch.zeros(1, 2, 64, device="cuda").half(), torch.ones(8, device="cuda")
    for kw in (dict(k=k.float(), v=k.float()), dict(v=k.bfloat16()), dict(k=k.cpu()), dict(k_cache=s["kc"].half()), dict(k_scale=s["ks"].half()),
               dict(k_scale=s["ks"][:, :, :1]), dict(v_scale=s["vs"].transpose(0, 2)), dict(slots=slots.long()), dict(slots=dev([1, 2])),
               dict(source=dev([0, 0])), dict(positions=slots), dict(inv_freq=one), dict(positions=slots, inv_freq=one[:4]),
               dict(positions=slots, inv_freq=torch.ones(40, device="cuda")), dict(interleaved=1), dict(rope_scale=math.inf),
               dict(q=half, source=dev([0])), dict(q=half.bfloat16()), dict(q=torch.zeros(2, 2, 64, device="cuda").half()),
               dict(k=k.clone().requires_grad_()), dict(slots=slots.cpu()), dict(k=k[..., :48], v=k[..., :48]), dict(err=slots.long())):
        with pytest.raises(ValueError):
            append(**kw)
    for kw in (dict(q=s["q"].float()), dict(q=s["q"][..., :32]), dict(k_cache=s["kc"][:, :, :1]), dict(scale=0.0), dict(scale=-1.0),
               dict(max_new=0), dict(max_new=D.MAX_NEW + 1), dict(window=-1), dict(sinks=-1), dict(lens=s["lens"].long()),
               dict(cu=s["cu"][:1]), dict(mask=dev([[1, 1]])[:, ::2].contiguous().long()), dict(positions=dev([1, 2])),
               dict(workspace=torch.zeros(100, dtype=torch.uint8, device="cuda")), dict(k_scale=torch.ones(s["ks"].shape[0], 3, 2, device="cuda"),
               v_scale=torch.ones(s["ks"].shape[0], 3, 2, device="cuda")), dict(max_new=40, mask=dev([[1]])), dict(table=s["table"].cpu())):
        with pytest.raises(ValueError):
            attention(**kw)
    with pytest.raises(ValueError):
        D.DraftCache8(1, 1, 4, 16, 64, 2, 64, block=12)
    with pytest.raises(ValueError):
        D.DraftCache8(1, 1, 4, 16, 64, 2, 96)
