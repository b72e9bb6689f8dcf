"""Token log-probabilities (hs_guard_b200.drafts.token_logprobs) on a B200 against 64-bit values.

Ids are equal. Tolerances: a thread adds up to c = vocab / 512 + 32 terms in fp32, each within 2^-22 (exponential) and
2^-23 |d| (its argument d, a difference to the row's largest over the temperature) of itself:
  log-sum-exp, log p   (c + 8) 2^-24 + 2^-22 (1 + E|d|) for ln S, E|d| the mean over p, + 2^-22 (|d_i| + |m| / T) for what it
                       is added to
  entropy              that, and as much times E|d| again for U / S: (1 + E|d|) ((c + 8) 2^-23 + 2^-22 (1 + E d^2 / max(E|d|, 1)))
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def D():
    from hs_guard_b200.build import build
    build()
    from hs_guard_b200 import drafts
    return drafts


def reference(x, given, top, temperature):
    z = x.double() / temperature
    m = z.amax(-1)
    z = z - m[:, None]  # 64 bits do not hold the logarithm of a sum beside the lowest fp32 number
    log_s = torch.log(torch.exp(z).sum(-1))
    lse = m + log_s
    p = torch.exp(z - log_s[:, None])
    entropy = -torch.special.xlogy(p, p).sum(-1)
    d = torch.where(p > 0, -z, 0.0)
    d1, d2 = (p * d).sum(-1), (p * d * d).sum(-1)
    given = given.long()
    lp = torch.where(given >= 0, z.gather(1, given.clamp(min=0)) - log_s[:, None], 0.0)
    ids = torch.sort(x.float(), dim=-1, descending=True, stable=True)[1][:, :top]
    c = x.shape[1] / 512 + 32
    base = (c + 8) * 2.0 ** -24 + 2.0 ** -22 * (1 + d1)
    tol = {"lse": base + 2.0 ** -22 * m.abs(),
           "entropy": (1 + d1) * ((c + 8) * 2.0 ** -23 + 2.0 ** -22 * (1 + d2 / d1.clamp(min=1)))}
    return lp, entropy, lse, z.gather(1, ids) - log_s[:, None], ids, base, tol, m


def check(got, x, given, top, temperature):
    lp, entropy, lse, tops, ids, base, tol, m = reference(x, given if given.dim() == 2 else given[:, None], top, temperature)
    if given.dim() == 1:
        lp = lp[:, 0]
    assert got.logprobs.shape == given.shape and got.top.shape == got.top_ids.shape == (x.shape[0], top)
    assert torch.equal(got.top_ids.long(), ids)

    def near(a, b, t):
        a = a.double()
        same = (a == b)  # infinities
        far = (a - b).abs()
        assert bool((same | (far <= t)).all()), float(torch.where(same, 0.0, far / t).max())

    near(got.lse, lse, tol["lse"])
    near(got.entropy, entropy, tol["entropy"])
    finite = lambda v: torch.where(torch.isfinite(v), v.abs(), 0.0)  # noqa: E731
    wide = base if lp.dim() == 1 else base[:, None]
    near(got.logprobs, lp, wide + 2.0 ** -22 * (1 + finite(lp) + (m.abs() if lp.dim() == 1 else m.abs()[:, None])))
    near(got.top, tops, base[:, None] + 2.0 ** -22 * (1 + finite(tops) + m.abs()[:, None]))


def logits(rows, vocab, dtype, seed, stride=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = 3 * torch.randn(rows, vocab + stride, generator=g, device="cuda")
    at = torch.randint(0, vocab, (rows, 5), generator=g, device="cuda")
    x.scatter_(1, at, 12 + 3 * torch.randn(rows, 5, generator=g, device="cuda"))
    x = x.to(dtype)[:, :vocab]
    given = torch.randint(0, vocab, (rows, 3), generator=g, device="cuda").int()
    given[:, 0] = at[:, 0].int()
    given[rows // 2, 1] = -1
    return x, given


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab,top,temperature,stride", [
    (1, 1, 1, 1.0, 0), (1, 3, 3, 1.0, 0), (3, 64, 64, 0.5, 1), (2, 65, 64, 1.0, 3), (5, 1000, 5, 2.0, 0), (1, 248320, 20, 1.0, 0),
    (7, 50001, 20, 0.7, 0), (40, 4097, 64, 1.0, 6), (333, 32001, 1, 1.0, 0), (600, 2049, 20, 1.3, 0), (130, 9999, 0, 1.0, 2)])
def test_logprobs(D, rows, vocab, top, temperature, stride, dtype):
    x, given = logits(rows, vocab, dtype, rows + vocab, stride)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(D.token_logprobs(x, given, top, temperature, err), x, given, top, temperature)
    assert int(err.item()) == 0
    flat = given[:, 0].contiguous()
    got = D.token_logprobs(x, flat, top, temperature)
    check(got, x, flat, top, temperature)
    again = D.token_logprobs(x, flat, top, temperature)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "steps", "lowest", "masked", "peak", "zeros"])
@pytest.mark.parametrize("rows,vocab", [(1, 30000), (400, 5001), (3, 700)])
def test_rows_that_are_hard_to_select_from(D, rows, vocab, kind, dtype):
    """Ties everywhere, sorted rows, rows of the type's lowest value, rows where almost everything is forbidden."""
    i = torch.arange(vocab, device="cuda").float().expand(rows, -1)
    low = torch.finfo(dtype).min
    x = {"equal": torch.full((rows, vocab), 2.5, device="cuda"), "rising": i / vocab * 20, "falling": -i / vocab * 20,
         "steps": torch.floor(i / 97) % 5, "lowest": torch.full((rows, vocab), low, device="cuda"),
         "masked": torch.where(i % 50 == 7, 1.0 - i / vocab, -math.inf), "peak": torch.where(i == 11, 90.0, -90.0),
         "zeros": torch.where(i % 2 == 0, 0.0, -0.0)}[kind].to(dtype).contiguous()
    top = 20 if kind != "masked" or vocab > 1000 else 14
    given = torch.full((rows, 1), 7, dtype=torch.int32, device="cuda")
    check(D.token_logprobs(x, given, top), x, given, top, 1.0)


def test_alternatives_that_are_forbidden(D):
    """Fewer allowed tokens than alternatives: -inf for the others, the lowest first."""
    x = torch.full((2, 5000), -math.inf, device="cuda")
    x[:, [4, 900, 4999]] = torch.tensor([1.0, 2.0, 1.0], device="cuda")
    got = D.token_logprobs(x, None, 6)
    assert got.logprobs.shape == (2, 0) and got.top_ids[0].tolist() == [900, 4, 4999, 0, 1, 2]
    assert bool(torch.isneginf(got.top[:, 3:]).all()) and bool(torch.isfinite(got.top[:, :3]).all())


def test_rows_without_a_distribution(D):
    x = torch.zeros(5, 3000, device="cuda")
    x[1] = -math.inf
    x[2, 77] = math.nan
    x[3, 2999] = math.inf
    given = torch.zeros(5, 1, dtype=torch.int32, device="cuda")
    got = D.token_logprobs(x, given, 4)
    for r in (1, 2, 3):
        assert bool(torch.isnan(got.logprobs[r]).all() and torch.isnan(got.top[r]).all() and torch.isnan(got.entropy[r]))
        assert got.top_ids[r].tolist() == [-1] * 4
    assert got.lse[1] == -math.inf and bool(torch.isnan(got.lse[2:4]).all())
    check(D.Logprobs(*(t[[0, 4]] for t in got)), x[[0, 4]], given[[0, 4]], 4, 1.0)


def test_tokens_beyond_the_vocabulary(D):
    x, given = logits(4, 500, BF16, 1)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    bad = given.clone()
    bad[1, 2] = 500
    got, want = D.token_logprobs(x, bad, 3, err=err), D.token_logprobs(x, given, 3)
    assert int(err.item()) == 4 and bool(torch.isnan(got.logprobs[1, 2]))
    same = torch.ones(4, 3, dtype=torch.bool)
    same[1, 2] = False
    assert torch.equal(got.logprobs[same], want.logprobs[same]) and torch.equal(got.top_ids, want.top_ids)


def test_no_rows_other_strides_streams_and_graphs(D):
    e = D.token_logprobs(torch.zeros(0, 10, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"), 2)
    assert [tuple(t.shape) for t in e] == [(0,), (0,), (0,), (0, 2), (0, 2)]
    x, given = logits(6, 7001, F16, 2)
    want = D.token_logprobs(x, given, 5)
    spread = torch.empty(6, 9003, dtype=F16, device="cuda")[:, 1:7002]
    spread.copy_(x)
    same = torch.as_strided(x.clone()[2], (6, 7001), (0, 1))
    check(D.token_logprobs(spread, given, 5), x, given, 5, 1.0)  # rows that begin elsewhere are summed in another order
    check(D.token_logprobs(same, given, 5), same, given, 5, 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = D.token_logprobs(x, given, 5)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    y = x.clone()
    with torch.cuda.graph(graph):
        got = D.token_logprobs(y, given, 5)
    y.copy_(x.flip(1))
    graph.replay()
    torch.cuda.synchronize()
    check(got, y, given, 5, 1.0)


def test_refusals(D):
    x, given = logits(4, 500, BF16, 3)
    for kw in (dict(logits=x.double()), dict(logits=x[0]), dict(logits=x.cpu()), dict(logits=x[:, ::2]), dict(given=given.long()),
               dict(given=given[:2]), dict(given=given[:, ::2]), dict(top=65), dict(top=-1), dict(top=501, logits=x), dict(temperature=0.0),
               dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=1e9), dict(logits=x[:, :3].contiguous(), top=4),
               dict(logits=x.float().requires_grad_()), dict(err=given), dict(top=2.5)):
        with pytest.raises(ValueError):
            D.token_logprobs(**{**dict(logits=x, given=given), **kw})
