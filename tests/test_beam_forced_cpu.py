"""Beams over shared prefixes, step by step, with the same choices: logits are those of beams that read their prefixes by themselves."""
import numpy as np
import pytest

from beam_forced import search, sharpen, worst
from vllm_ascend_b200 import LLM, ops


def _llm():
    return sharpen(LLM("tiny-qwen", device="cpu", seed=1, block_size=16, max_model_len=128, max_num_seqs=16))


def _prompts(*lengths):
    rng = np.random.default_rng(6)
    return [rng.integers(1, 500, size=n).tolist() for n in lengths]


def _slack(row):
    # 32 bits all the way: some hundred roundings of half a step, 2^-24, of numbers of the logits' size
    return 2.0 ** -24 * 400 * row.abs().max()


@pytest.mark.parametrize("lengths", [(33, 20, 48), (64,)])
def test_same_logits_in_every_step(monkeypatch, lengths):
    alone, choices = search(_llm(), monkeypatch, _prompts(*lengths), 3, 20, False)
    shared, _ = search(_llm(), monkeypatch, _prompts(*lengths), 3, 20, True, choices)
    assert worst(alone, shared, _slack) < 1


def _rough(row):
    # what the same comparison allows in bf16
    return 0.15 * row.std() + 2.0 ** -8 * row.abs().max()


def test_what_the_comparison_shows(monkeypatch):
    """Partly filled pages that do not follow their beams, and a prefix read through another group's pages, are far outside of what bf16 may be off by."""
    prompts = _prompts(33, 36)
    alone, choices = search(_llm(), monkeypatch, prompts, 3, 20, False)
    with monkeypatch.context() as m:
        m.setattr(ops, "reorder_beams", lambda *a: None)
        assert worst(alone, search(_llm(), monkeypatch, prompts, 3, 20, True, choices)[0], _rough) > 2
    plan = ops.plan_shared_prefix
    with monkeypatch.context() as m:
        m.setattr(ops, "plan_shared_prefix", lambda meta, starts, *a: plan(meta, starts.masked_fill(starts > 0, meta.num_reqs), *a))
        assert worst(alone, search(_llm(), monkeypatch, prompts, 3, 20, True, choices)[0], _rough) > 2
