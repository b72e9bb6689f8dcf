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
