"""Draft scoring on a B200 where it can go wrong: weights far below the largest one, tokens of no request, rings without
room, page ids outside their range, caches used on several streams, gradients, and the widest shapes.

Tolerances are those of test_gpu_drafts.py unless a test says otherwise; all were derived before the first run."""
import math

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
