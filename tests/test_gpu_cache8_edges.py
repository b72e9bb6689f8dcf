"""The 8-bit cache on a B200 where it can go wrong: slot lists that do not ascend or are mostly padding, sums beyond fp32, pages
outside the cache, positions that repeat, V of zeros over long caches, outliers in queries, chunks beside single tokens.

Tolerances are those of test_gpu_cache8.py unless a test says otherwise; all were derived before the first run."""
import math

import pytest
import torch

from test_gpu_cache8 import (BF16, D, F16, F8, U, append_reference, append_state, attend, attention_reference, attention_state,  # noqa: F401
                             check_append, check_attention, dev, err_word, pool, turned)

pytestmark = pytest.mark.gpu


# ---- append_8bit: lists that are wrong, lists of padding --------------------------------------------------------------
@pytest.mark.parametrize("slots,good", [
    ([5, 4, 6, 7], [0, 2, 3]), ([5, 5, 6], [0, 2]), ([5, 4, 5, 6], [0, 3]), ([0, 3, 2, 4, 1, 9, 15, 15, 3, 16, 17], [0, 1, 3, 5, 6, 9, 10]),
    ([20, 16, 17, 21, 32, 33, 32, 40], [0, 3, 4, 5, 7]), ([9, 3, -1, 10, -1, -1, 8, -1, 12, 13], [0, 3, 8, 9]),
    ([0, 1] + [0] * 70 + [2, 3], [0, 1, 72, 73]), ([0, -1] + [-1] * 300 + [0] + [-1] * 3000 + [7, 8, 7, 9], [0, 3303, 3304, 3306])])
def test_append_skips_only_the_slots_that_do_not_ascend(D, slots, good):
    """Of a block's entries those that stand above all before them are written, whatever is between them."""
    page, hkv, dim, n = 16, 2, 64, len(slots)
    g = torch.Generator().manual_seed(n)
    k = torch.randn(n, hkv, dim, generator=g)
    k[0] *= 16  # the first entries' scale holds for all: no code is rounded twice
    k[[i for i in good if slots[i] % 16 == 0]] *= 16
    k = k.half().cuda()
    s = append_state(4, page, 16, hkv, dim, False, 30)
    if slots[0] % 16:
        s["ks"][0], s["vs"][0], s["ks"][1], s["vs"][1] = 1.0, 1.0, 1.0, 1.0
    kept = [x if i in good else -1 for i, x in enumerate(slots)]
    ref = append_reference(s, k, k, kept, None, torch.zeros(n), torch.zeros(0), False, 1.0)
    err = err_word()
    D.append_8bit(k, k, s["kc"], s["vc"], s["ks"], s["vs"], dev(slots), err=err)
    assert int(err.item()) == 3
    check_append(s, ref, False)


@pytest.mark.parametrize("gap", [31, 1000, 4095, 4096, 5000, 20000])
def test_append_over_long_padding(D, gap):
    """Entries far apart in a padded list: runs that go on behind the padding, and ones that begin there."""
    page, hkv, dim = 64, 2, 64
    slots = [-1] * gap + [64, 65] + [-1] * gap + [66, 67, 96] + [-1] * gap + [130] + [-1] * gap + [131, 192] + [-1] * gap
    n = len(slots)
    k = torch.randn(n, hkv, dim, generator=torch.Generator().manual_seed(gap)).bfloat16().cuda()
    s = append_state(5, page, 32, hkv, dim, False, 31)
    at = [i for i, x in enumerate(slots) if x >= 0]
    ref = append_reference(s, k[at], k[at], [slots[i] for i in at], None, torch.zeros(len(at)), torch.zeros(0), False, 1.0)
    err = err_word()
    D.append_8bit(k, k, s["kc"], s["vc"], s["ks"], s["vs"], dev(slots), err=err)
    assert int(err.item()) == 0
    check_append(s, ref, False)


def test_append_time_goes_by_tokens_not_by_padding(D):
    """Ten tokens in a list of 2^17 entries, as a captured call with room for many has them: tens of us more than in one of 16. Where
    every block of padding looked for the entry before it, they took 3,650."""
    page, hkv, dim, n = 64, 2, 64, 1 << 17
    s = append_state(2, page, 64, hkv, dim, False, 32)
    k = torch.randn(n, hkv, dim, device="cuda").half()

    def us(slots):
        times = []
        for _ in range(12):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            D.append_8bit(k, k, s["kc"], s["vc"], s["ks"], s["vs"], slots)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b) * 1e3)
        return sorted(times)[4]

    few = dev(list(range(10)) + [-1] * 6)
    for where in (0, n // 2, n - 10):
        many = torch.full((n,), -1, dtype=torch.int32, device="cuda")
        many[where:where + 10] = torch.arange(10, device="cuda")
        assert us(many) < us(few) + 200, where


def test_append_pairs_whose_sum_is_beyond_fp32(D):
    """Two finite elements that turn together and whose magnitudes add up to more than fp32 has count as the largest number, not as
    infinite ones, which count for nothing."""
    page, dim = 16, 64
    k = torch.zeros(4, 1, dim)
    k[0, 0, 3], k[0, 0, 3 + 32] = 2e38, -3e38
    k[1, 0, 3], k[1, 0, 3 + 32], k[1, 0, 5] = 2e38, math.inf, 1.0
    k[2, 0, 4], k[2, 0, 4 + 32], k[2, 0, 5] = 3e38, 3e38, math.nan
    k[3, 0, 7] = 1.0
    k = k.bfloat16().cuda()
    s = append_state(5, page, 16, 1, dim, False, 33)
    p = torch.zeros(4, dtype=torch.int32, device="cuda")
    D.append_8bit(k, k, s["kc"], s["vc"], s["ks"], s["vs"], dev([0, 16, 32, 48]), positions=p, inv_freq=torch.ones(32, device="cuda"))
    assert s["ks"][:4, 0, 0].tolist() == [2.0 ** 120, 2.0 ** -8, 2.0 ** 120, 2.0 ** -8]
    got, x = s["kc"][:4, 0, 0].double() * s["ks"][:4, 0].double(), k[:, 0].double()
    for r, d in ((0, 3), (0, 35), (2, 4), (2, 36), (1, 5), (3, 7)):
        assert abs(float(got[r, d] - x[r, d])) <= 2.0 ** -4 * abs(float(x[r, d]))
    assert bool(torch.isnan(got[1, [3, 35]]).all()) and bool(torch.isnan(got[2, [5, 37]]).all())


# ---- attention_8bit ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,hq,hkv,page,block,heads_first", [(64, 4, 2, 16, 16, False), (64, 4, 2, 8, 8, True), (128, 8, 2, 32, 8, False),
                                                               (128, 8, 2, 128, 32, True), (256, 8, 2, 16, 8, False), (256, 8, 2, 64, 64, True)])
@pytest.mark.parametrize("n", [1, 3, 40])
@pytest.mark.parametrize("bad", [-1, 1 << 20])
def test_attention_skips_pages_outside_the_cache(D, dim, hq, hkv, page, block, heads_first, n, bad, dtype):
    """Tokens of a page that the cache does not have are not seen, as if the request were without them: shared memory that holds
    NaN from another call does not show."""
    lens = [20 * page + 3, 9 * page, 11 * page + page // 2]
    lens = [x + n for x in lens]
    s = attention_state(dim, hq, hkv, page, block, lens, [n] * 3, dtype, heads_first, seed=40 + n)
    nan = dict(s, kc=pool(s["kc"].shape[0], page, hkv, dim, heads_first, fill=0x7f), vc=pool(s["kc"].shape[0], page, hkv, dim, heads_first, fill=0x7f))
    wrong, without = dict(s, table=s["table"].clone()), dict(s, table=s["table"].clone(), lens=s["lens"].clone())
    for b, pages in ((0, (3, 4, 11)), (2, (0,))):
        for p in pages:
            wrong["table"][b, p] = bad
        rest = [x for i, x in enumerate(s["table"][b].tolist()) if i not in pages]
        without["table"][b] = dev(rest + [-7] * len(pages))
        without["lens"][b] -= len(pages) * page
    ref = attention_reference(without, dim ** -0.5)
    for _ in range(3):
        attend(D, nan, dim ** -0.5, n)
        err = err_word()
        got = attend(D, wrong, dim ** -0.5, n, err=err)
        assert int(err.item()) == 6
        check_attention(got, ref, dtype)


def test_attention_of_a_request_without_a_page(D):
    """Every page outside the cache: nothing is seen."""
    for n in (1, 40):
        s = attention_state(128, 8, 2, 16, 16, [50, 60], [n, n], F16, seed=45)
        good = attention_reference(s, 0.1)
        s["table"][0] = -1
        out, lse = attend(D, s, 0.1, n)
        assert bool((out[:n] == 0).all()) and bool(torch.isneginf(lse[:n]).all())
        check_attention((out[n:], lse[n:]), [x[n:] for x in good], F16)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,hq,hkv", [(64, 4, 4), (128, 4, 2), (256, 2, 1)])
@pytest.mark.parametrize("lens,counts", [([420, 33, 1, 60, 60, 60, 60, 60, 60, 60], [150, 1, 1, 1, 1, 1, 1, 1, 1, 1]), ([700, 500], [600, 300])])
@pytest.mark.parametrize("step,window,sinks", [(0.125, 10, 0), (0.125, 10, 300), (0.02, 5, 2), (3, 40, 0)])
def test_attention_positions_without_a_mask(D, lens, counts, dim, hq, hkv, step, window, sinks, dtype):
    """A chain whose positions repeat (parts of a picture, say) or leave some out: the window goes by them, not by the places."""
    s = attention_state(dim, hq, hkv, 16, 16, lens, counts, dtype, seed=46)
    s["positions"] = dev([n - c + int(t * step) for n, c in zip(lens, counts) for t in range(c)])
    err = err_word()
    got = attend(D, s, dim ** -0.5, max(counts), window=window, sinks=sinks, err=err)
    assert int(err.item()) == 0
    check_attention(got, attention_reference(s, dim ** -0.5, window, sinks), dtype)


@pytest.mark.parametrize("n", [1, 24])
@pytest.mark.parametrize("values", ["zeros", "some"])
def test_attention_over_many_values_of_zero(D, n, values):
    """Blocks of zeros have the smallest scale there is: the sum of the weights over it stays a number, over 150,000 keys too."""
    page, dim, keys = 128, 64, 150000
    pages = -(-keys // page)
    k, v = (torch.zeros(pages, page, 1, dim, dtype=torch.uint8, device="cuda").view(F8) for _ in range(2))
    ks, vs = torch.ones(pages, 1, 1, device="cuda"), torch.full((pages, 1, 1), 2.0 ** -100, device="cuda")
    share = 0.0
    if values == "some":  # a page of ones
        v.view(torch.uint8)[7] = 0x38
        vs[7] = 1.0
        share = page / keys
    q = torch.zeros(n, 1, dim, device="cuda").half()
    table = torch.arange(pages, device="cuda").int()[None]
    mask = torch.full((n, 1), -1, dtype=torch.int32, device="cuda")  # all of them see all
    out, lse = D.attention_8bit(q, k, v, ks, vs, table, dev([keys]), dev([0, n]), 0.125, n, mask=mask)
    more = (keys / 8 + 32) * 2.0 ** -23
    assert float((lse.double() - math.log(keys)).abs().max()) <= more + 4e-6 * (1 + math.log(keys))
    assert float((out.double() - share).abs().max()) <= (U[F16] + 2.0 ** -11 + more) * share + 2.0 ** -25


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("largest", [230.0, 447.0])
def test_attention_queries_with_an_outlier(D, dim, dtype, largest):
    """One element of a query hundreds of times the others, over keys that are small there, so that the others decide.

    For many rows a query is a sum of e4m3 numbers, its largest element brought to (224, 448], e4m3's last step there 2^-9: an
    element is off by at most 2^-10 / 224 of the largest. Scores by that times scale sum |k| more than otherwise, twice in a weight."""
    n = 40
    s = attention_state(dim, 4, 2, 16, 16, [500, 300], [n, n], dtype, seed=47)
    q = torch.empty(2 * n, 4, dim, device="cuda").uniform_(-1.5, 1.5, generator=torch.Generator(device="cuda").manual_seed(1))
    q[..., 5] = largest
    s["q"] = q.to(dtype)
    s["kc"].view(torch.uint8)[:, :, :, 5] = torch.where(torch.isnan(s["kc"][:, :, :, 5].float()), 0x7f, 0).to(torch.uint8)
    scale = 0.02
    out, lse, tol, ltol = attention_reference(s, scale)
    keys = torch.where(torch.isnan(s["ks"]), 0.0, s["ks"])[..., None].repeat_interleave(16, 1)[..., 0]
    sums = (torch.nan_to_num(s["kc"].float()).abs().sum(-1) * keys).max()
    ds = scale * 2.0 ** -10 / 224 * largest * float(sums)
    most = torch.nan_to_num(s["vc"].float()).abs().mul(torch.nan_to_num(s["vs"]).repeat_interleave(16, 1)[..., None]).max()
    check_attention(attend(D, s, scale, n), (out, lse, tol + 2 * ds * float(most), ltol + ds), dtype)


@pytest.mark.parametrize("singles", [9, 300])
def test_attention_of_a_chunk_beside_single_tokens(D, singles):
    """A prompt's chunk first, in the middle and last among requests of one token, in one call."""
    for at in (0, singles // 2, singles):
        lens, counts = [31 + 7 * (i % 40) for i in range(singles)], [1] * singles
        lens.insert(at, 900)
        counts.insert(at, 700)
        s = attention_state(128, 8, 2, 16, 16, lens, counts, BF16, seed=48)
        check_attention(attend(D, s, 0.09, 700), attention_reference(s, 0.09), BF16)
