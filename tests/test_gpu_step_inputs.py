"""Host buffers of a step's inputs on the GPU: steps that nobody waits for, on a device that is late."""
import numpy as np
import pytest
import torch

from vllm_ascend_b200 import LLM, SamplingParams
from vllm_ascend_b200.config import ModelConfig

pytestmark = pytest.mark.gpu


def _llm(max_num_batched_tokens=256, **kw):
    cfg = ModelConfig(name="portions", architecture="Qwen3ForCausalLM", vocab_size=2048, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, head_dim=64, qk_norm=True, rope_theta=1e6, dtype="float32")
    return LLM(cfg, device="cuda", max_model_len=2048, max_num_seqs=8, max_num_batched_tokens=max_num_batched_tokens, num_gpu_blocks_override=200, block_size=64,
               enforce_eager=True, seed=2, **kw)


def _prompts(*lengths):
    rng = np.random.default_rng(11)
    return [rng.integers(1, 2000, size=n).tolist() for n in lengths]


def _pace(llm, monkeypatch, late):
    """Every pass begins 20 ms late (the host is then several steps ahead), or the host waits for it."""
    runner = llm.engine.runner
    forward = runner._forward

    def paced(T, meta):
        if late:
            torch.cuda._sleep(40_000_000)
        out = forward(T, meta)
        if not late:
            torch.cuda.synchronize()
        return out
    monkeypatch.setattr(runner, "_forward", paced)
    return llm


@pytest.mark.parametrize("caching", [False, True])
def test_beams_of_prompts_in_many_portions(monkeypatch, caching):
    prompts, outs = _prompts(1500, 300), []
    for late in (False, True):
        llm = _pace(_llm(enable_prefix_caching=caching), monkeypatch, late)
        # a second time from the prefix cache
        outs.append([llm.beam_search(p, beam_width=3, max_tokens=4, ignore_eos=True) for p in (prompts, [q + [5] for q in prompts])])
    assert outs[0] == outs[1]


def test_portions_and_whole_prompts_agree():
    """Six portions and one: the same scores but for roundings of 32 bits (1e-3 of four tokens' log-probabilities, around 8 each)."""
    prompts = _prompts(1500)
    found = [_llm(max_num_batched_tokens=n).beam_search(prompts, beam_width=3, max_tokens=4, ignore_eos=True)[0] for n in (256, 2048)]
    np.testing.assert_allclose(*[[b["cum_logprob"] for b in best] for best in found], atol=1e-3)


@pytest.mark.parametrize("asynchronous", [False, True])
def test_prompts_in_many_portions(monkeypatch, asynchronous):
    outs = []
    for late in (False, True):
        llm = _pace(_llm(async_scheduling=asynchronous), monkeypatch, late)
        sp = SamplingParams(temperature=0.0, max_tokens=5, ignore_eos=True, logprobs=0)
        outs.append([(o.outputs[0].token_ids, o.outputs[0].logprobs) for o in llm.generate(_prompts(1500, 300), sp)])
    assert outs[0] == outs[1]
