"""Log-probabilities of beams keep 64 bits from round to round."""
import math

import numpy as np
import pytest
import torch

from beam_cases import totals
from vllm_ascend_b200 import LLM, ops


def test_selection_in_64_bits():
    g = torch.Generator().manual_seed(4)
    logits, scores = torch.randn(6, 203, generator=g), -torch.rand((2, 3), generator=g, dtype=torch.float64) * 300
    scores[1, 2] = -math.inf
    values, parents, tokens = ops.beam_select(logits, scores, 7, dtype=torch.float64)
    want, at = torch.sort(totals(logits, scores), dim=-1, descending=True, stable=True)
    assert values.dtype == torch.float64 and parents.dtype == torch.int32 and tokens.dtype == torch.int64
    assert torch.equal(parents.long() * 203 + tokens, at[:, :7])
    # half a step of 64 bits each for the logarithm of the sum, its difference from a logit and the sum with a score below 512
    assert ((values - want[:, :7]).abs() <= 2 * 3 * 512 * 2.0 ** -53).all()
    near = torch.tensor([[-100.0, -100.0 + 1e-9]], dtype=torch.float64)
    assert ops.beam_select(logits[:1].expand(2, -1), near, 1, dtype=torch.float64)[1].item() == 1


def test_types_of_scores():
    logits, scores = torch.zeros(6, 5), torch.zeros(2, 3)
    for x, kw in ((scores, {"dtype": torch.float64}), (scores.double(), {}), (scores.double(), {"dtype": torch.float32}),
                  (scores.half(), {"dtype": torch.float16}), (scores.long(), {"dtype": torch.int64})):
        with pytest.raises(ValueError):
            ops.beam_select(logits, x, 2, **kw)
    assert ops.beam_select(logits, scores, 2, dtype=torch.float32)[0].dtype == torch.float32


@pytest.mark.parametrize("width", [1, 4])
def test_long_answers_add_up(monkeypatch, width):
    """A model whose logits are the same for all beams of a round: the best answer takes the best token each time."""
    rounds = 200
    llm = LLM("tiny-qwen", device="cpu", seed=1, block_size=16, max_model_len=256, max_num_seqs=8)
    vocab = llm.engine.cfg.model.vocab_size
    g = torch.Generator().manual_seed(9)
    table, at = torch.randn(rounds, vocab, generator=g), iter(range(rounds))

    def logits(so, rows=None):
        return table[next(at)].expand(len(rows) if rows is not None else so.num_scheduled_tokens, -1)
    monkeypatch.setattr(llm.engine.runner, "device_logits", logits)
    best = llm.beam_search([[1, 2, 3]], beam_width=width, max_tokens=rounds, ignore_eos=True)[0]
    lp = torch.log_softmax(table.double(), -1)
    top = lp.sort(-1, descending=True)[0]
    assert best[0]["tokens"] == lp.argmax(-1).tolist()
    # sums of 200 numbers of 64 bits, below 2048 in all: half a step each, in either form
    assert abs(best[0]["cum_logprob"] - float(top[:, 0].sum())) <= 4 * rounds * 2048 * 2.0 ** -53
    # answers one token away from the best, by what that costs
    costs = np.sort((top[:, :1] - top[:, 1:width + 1]).reshape(-1).numpy())
    for b, cost in zip(best[1:2], costs):
        assert abs(b["cum_logprob"] - (float(top[:, 0].sum()) - cost)) <= 8 * rounds * 2048 * 2.0 ** -53
