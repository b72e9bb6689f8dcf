"""Draft scoring beside a live engine on a B200: the engine's own rings as a cache, its own ring attention as the measure
for chains, and the example that runs the whole path.

Tolerances: fp16 results of values around 1 against 64 bits: 2^-11 (|o| + sum p |v|) with |v| up to 5, below 5e-3."""
import os
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CONTEXTS = [700, 41, 513, 64]


@pytest.fixture(scope="module")
def example():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import score_drafts
    finally:
        sys.path.pop(0)
    return score_drafts


@pytest.fixture(scope="module")
def engine(weights_seed0):
    from hs_guard_b200.build import build
    from hs_guard_b200.engine import SlotEngine
    build()
    eng = SlotEngine(weights_seed0, 4)
    rng = np.random.default_rng(5)
    eng.step([(s, rng.integers(0, 1000, n).tolist()) for s, n in enumerate(CONTEXTS)])
    yield eng
    eng.close()


def layer_of(example, engine, index=0):
    where = [i for i, t in enumerate(engine.cfg.layer_types) if t == "full_attention"][index]
    return example.Layer(engine.weights["layers"][where], engine.weights["inv_freq"])


@pytest.mark.parametrize("index,slots,sizes", [(0, [2, 0, 3], [12, 7, 15]), (5, [1], [1]), (3, [0, 1, 2, 3], [1, 40, 3, 33])])
def test_trees_over_live_rings(example, engine, index, slots, sizes):
    before = [engine.pools()[n].clone() for n in ("ring_k", "ring_v", "ring_pos")]
    worst, _ = example.over_rings(engine, layer_of(example, engine, index), slots, sizes, seed=index, layer_index=index)
    assert worst < 5e-3
    torch.cuda.synchronize()
    for n, t in zip(("ring_k", "ring_v", "ring_pos"), before):
        assert torch.equal(engine.pools()[n], t), "scoring drafts must leave the conversation as it is"


def test_chains_over_live_rings_match_ring_attention(engine):
    """A chain of drafted tokens is a tick's own tokens: the engine's ring attention gives the same, to fp16 rounding."""
    from hs_guard_b200 import _lib, drafts
    lb, slots = 8, [0, 1, 2, 3]
    n, g = len(slots), torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(n, lb, 8, 256, generator=g, device="cuda").half()
    k, v = (torch.randn(n, lb, 2, 256, generator=g, device="cuda").half() for _ in range(2))
    k_cache, v_cache, table, lens = drafts.ring_cache(engine, 1, slots)
    cu = torch.arange(0, n * lb + 1, lb, dtype=torch.int32, device="cuda")
    out, _ = drafts.tree_attention(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), k_cache, v_cache, table, lens, cu,
                                   1.0 / 16, lb, window=512)
    pools = engine.pools()
    grouped = q.float().view(n, lb, 2, 4, 256).permute(0, 2, 3, 1, 4).reshape(n, 2, 4 * lb, 256).contiguous()
    ref = torch.empty_like(grouped)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    i64 = dict(dtype=torch.int64, device="cuda")
    new_k, new_v = (x.transpose(1, 2).contiguous() for x in (k, v))
    args = [torch.tensor(slots, **i64), lens.long(), torch.full((n,), lb, **i64)]
    _lib.check(_lib.lib().hsg_ring_attention(
        grouped.data_ptr(), pools["ring_k"][1].data_ptr(), pools["ring_v"][1].data_ptr(), new_k.data_ptr(),
        new_v.data_ptr(), pools["ring_pos"].data_ptr(), *(a.data_ptr() for a in args), n, lb, engine.max_slots, 1.0 / 16,
        ref.data_ptr(), 0, err.data_ptr(), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    ref = ref.view(n, 2, 4, lb, 256).permute(0, 3, 1, 2, 4).reshape(n * lb, 8, 256)
    torch.testing.assert_close(out.float(), ref, rtol=2e-3, atol=5e-3)


def test_ring_cache_refusals(engine):
    from hs_guard_b200 import drafts
    for layer, slots in ((6, [0]), (-1, [0]), (0, [4]), (0, [-1]), (0, [])):
        with pytest.raises(ValueError):
            drafts.ring_cache(engine, layer, slots)


def test_pages_accept_branches(example, engine):
    worst, lens = example.over_pages(layer_of(example, engine), [300, 17, 1200], [9, 5, 16], 3)
    assert worst < 5e-3 and all(a > b for a, b in zip(lens, [300, 17, 1200]))
