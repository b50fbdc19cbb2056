"""Log-probabilities of beams keep 64 bits from round to round, on the GPU."""
import math

import pytest
import torch

from beam_cases import check_select, slack, totals
from vllm_ascend_b200 import LLM, ops

pytestmark = pytest.mark.gpu


def _some(rows, vocab, seed):
    """Rows of some elements at 0, the others at -inf: sums of exponentials are whole numbers."""
    g = torch.Generator().manual_seed(seed)
    n = torch.randint(1, vocab, (rows,), generator=g)
    order = torch.rand((rows, vocab), generator=g).argsort(-1)
    return torch.where(order < n[:, None], 0.0, -math.inf), n


@pytest.mark.parametrize("groups,width,vocab,k", [(1, 1, 1, 1), (1, 4, 32000, 8), (3, 5, 50257, 10), (2, 16, 20011, 256), (40, 8, 5003, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_selection_in_64_bits(groups, width, vocab, k, dtype):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = torch.empty((groups * width, vocab), device="cuda").normal_(std=2.5, generator=g).to(dtype)
    scores = -torch.rand((groups, width), device="cuda", generator=g, dtype=torch.float64) * 300
    if groups > 1:
        scores[0, 1], scores[1, 0] = -math.inf, math.nan
    values, parents, tokens = ops.beam_select(logits, scores, k, dtype=torch.float64)
    assert values.dtype == torch.float64
    mine = totals(logits, scores).gather(1, parents.long().cpu() * vocab + tokens.cpu())
    assert torch.equal(mine.isfinite(), values.isfinite().cpu())
    assert ((values.cpu() - mine).abs()[mine.isfinite()] <= slack(logits) + 1e-12).all()
    short = scores.float()                               # the same continuations, rounded once
    check_select(ops.beam_select(logits, short, k), logits, short, k)
    a, b = ops.beam_select(logits, short, k), ops.beam_select(logits, short.double(), k, dtype=torch.float64)
    assert torch.equal(a[0], b[0].float()) and torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])


def test_scores_that_32_bits_do_not_tell_apart():
    logits, _ = _some(2, 1000, 1)
    logits = logits[:1].expand(2, -1).cuda()
    for first in (0, 1):
        scores = torch.full((1, 2), -100.0, dtype=torch.float64, device="cuda")
        scores[0, first] += 1e-9
        _, parents, _ = ops.beam_select(logits, scores, 1, dtype=torch.float64)
        assert parents.item() == first


def test_rounds_add_up():
    rows, n = _some(300, 4099, 2)
    rows, want = rows.cuda(), 0.0
    scores = torch.zeros((1, 1), dtype=torch.float64, device="cuda")
    for i in range(300):
        scores, _, _ = ops.beam_select(rows[i:i + 1], scores, 1, dtype=torch.float64)
        want -= math.log(int(n[i]))
    # 300 sums and logarithms below 4096: half a step of 64 bits each, two on either side
    assert abs(scores.item() - want) <= 4 * 300 * 4096 * 2.0 ** -53


def test_long_answers_add_up(monkeypatch):
    llm = LLM("tiny-qwen", device="cuda", seed=1, block_size=16, max_model_len=256, max_num_seqs=8, num_gpu_blocks_override=64, enforce_eager=True)
    vocab, rounds = llm.engine.cfg.model.vocab_size, 200
    rows, n = _some(rounds, vocab, 3)
    rows, at = rows.cuda(), iter(range(rounds))
    monkeypatch.setattr(llm.engine.runner, "device_logits",
                        lambda so, rs=None: rows[next(at)].expand(len(rs) if rs is not None else so.num_scheduled_tokens, -1))
    best = llm.beam_search([[1, 2, 3]], beam_width=2, max_tokens=rounds, ignore_eos=True)[0]
    want = -sum(math.log(int(x)) for x in n)
    # all continuations of a round cost the same
    assert all(abs(b["cum_logprob"] - want) <= 4 * rounds * 4096 * 2.0 ** -53 for b in best)
