"""Beams over shared prefixes on the GPU, step by step, with the same choices: logits, and log-probabilities of all beams' tokens."""
import numpy as np
import pytest

from beam_forced import search, sharpen, worst
from vllm_ascend_b200 import LLM, SamplingParams
from vllm_ascend_b200.config import ModelConfig

pytestmark = pytest.mark.gpu


def _llm(**kw):
    cfg = ModelConfig(name="beams", architecture="Qwen3ForCausalLM", vocab_size=2048, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
                      num_attention_heads=8, num_key_value_heads=2, head_dim=128, qk_norm=True, rope_theta=1e6, dtype="bfloat16")
    return sharpen(LLM(cfg, device="cuda", max_model_len=1024, max_num_seqs=24, max_num_batched_tokens=1024, num_gpu_blocks_override=200, block_size=64,
                       cudagraph_capture_sizes=[1, 2, 4, 8, 16, 24], seed=5, **kw))


def _prompts(*lengths):
    rng = np.random.default_rng(6)
    return [rng.integers(1, 2000, size=n).tolist() for n in lengths]


def _slack(row):
    """Two layers round to bf16 some twenty times on either side, each by half a step at most, 2^-9 of the size: independent, 2^-9 sqrt(40 / 3) of the logits'
    spread, 0.007, and six times that for the largest of some 10^5 logits; four times as much for the second layer's scores, up to 8 in size,
    whose queries have been rounded.  And the logits' own, half a step each."""
    return 0.15 * row.std() + 2.0 ** -8 * row.abs().max()


@pytest.mark.parametrize("lengths", [(65, 100, 190), (64,), (700, 130, 66, 129)])
def test_same_logits_in_every_step(monkeypatch, lengths):
    prompts = _prompts(*lengths)
    alone, choices = search(_llm(), monkeypatch, prompts, 4, 24, False)
    llm = _llm()
    shared, _ = search(llm, monkeypatch, prompts, 4, 24, True, choices)
    assert any(k[1] == "shared" for k in llm.engine.runner.graphs) and len(shared) == 24
    assert worst(alone, shared, _slack) < 1


def _answers(choices, group, width):
    """(tokens, their log-probabilities) of a group's beams, from the choices of all rounds; no beam ends."""
    beams = [([], [], 0.0)]
    for totals, parents, tokens in choices:
        beams = [(beams[p][0] + [t], beams[p][1] + [total - beams[p][2]], total)
                 for total, p, t in zip(totals[group, :width].tolist(), parents[group, :width].tolist(), tokens[group, :width].tolist())]
    return [b[:2] for b in beams]


@pytest.mark.parametrize("share", [False, True])
def test_every_token_is_scored_as_in_a_prompt(monkeypatch, share):
    llm, prompts = _llm(), _prompts(200, 129, 66)
    seen, choices = search(llm, monkeypatch, prompts, 4, 24, share)
    slack = max(float(_slack(r)) for x in seen for r in x)
    for g, p in enumerate(prompts):
        answers = _answers(choices, g, 4)
        assert len({tuple(t) for t, _ in answers}) == 4
        for tokens, scores in answers:
            o = llm.generate([p + tokens], SamplingParams(temperature=0.0, max_tokens=1, prompt_logprobs=0))
            mine = [lp[t] for lp, t in zip(o[0].prompt_logprobs[len(p):], tokens)]
            # the token's own logit and the sum's logarithm
            np.testing.assert_allclose(scores, mine, atol=2 * slack)
