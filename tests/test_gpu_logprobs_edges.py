"""token_logprobs on a B200 where the alternatives' selection is hard for many rows, which blocks of fewer threads take.

Ids are equal and tolerances those of test_gpu_logprobs.py: a block of 256 threads adds two terms at a time, so that a thread's
sums take vocab / 512 steps there too."""
import math

import pytest
import torch

from test_gpu_logprobs import BF16, D, F16, F32, check, logits  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [592, 2500])
@pytest.mark.parametrize("vocab,top", [(255, 64), (256, 64), (257, 64), (384, 50), (384, 64), (400, 64), (512, 64), (513, 64), (512, 1)])
def test_small_vocabularies_of_many_rows(D, rows, vocab, top, dtype):
    """Fewer pieces than threads, and fewer of those than alternatives: every value is a candidate."""
    x, given = logits(rows, vocab, dtype, rows + vocab)
    check(D.token_logprobs(x, given, top), x, given, top, 1.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [3, 400, 600])
@pytest.mark.parametrize("allowed,top", [(10, 36), (255, 64), (300, 36), (300, 50), (500, 64), (512, 64), (520, 64)])
def test_a_run_of_allowed_tokens(D, rows, allowed, top, dtype):
    """A grammar that leaves a run of ids: a few threads have all the candidates."""
    vocab = 32000
    g = torch.Generator(device="cuda").manual_seed(allowed)
    x = torch.full((rows, vocab), -math.inf, device="cuda")
    x[:, 9000:9000 + allowed] = 10 + 10 * torch.rand(rows, allowed, generator=g, device="cuda")
    x = x.to(dtype)
    given = torch.randint(9000, 9000 + allowed, (rows, 2), generator=g, device="cuda").int()
    check(D.token_logprobs(x, given, top), x, given, top, 1.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "steps", "lowest", "masked", "peak", "zeros"])
@pytest.mark.parametrize("rows,vocab,top", [(600, 700, 14), (600, 1300, 20), (2500, 1300, 64), (600, 5001, 50)])
def test_many_rows_that_are_hard_to_select_from(D, rows, vocab, top, kind, dtype):
    """Hundreds of values tied at the last alternative's, sorted rows, rows where almost everything is forbidden."""
    i = torch.arange(vocab, device="cuda").float().expand(rows, -1)
    low = torch.finfo(dtype).min
    x = {"equal": torch.full((rows, vocab), 2.5, device="cuda"), "rising": i / vocab * 20, "falling": -i / vocab * 20,
         "steps": torch.floor(i / 97) % 5, "lowest": torch.full((rows, vocab), low, device="cuda"),
         "masked": torch.where(i % 50 == 7, 1.0 - i / vocab, -math.inf), "peak": torch.where(i == 11, 90.0, -90.0),
         "zeros": torch.where(i % 2 == 0, 0.0, -0.0)}[kind].to(dtype).contiguous()
    given = torch.full((rows, 1), 7, dtype=torch.int32, device="cuda")
    check(D.token_logprobs(x, given, top), x, given, top, 1.0)
