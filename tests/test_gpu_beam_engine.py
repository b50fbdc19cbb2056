"""Beam search and decode batches with a common prefix through the engine, on the GPU."""
import numpy as np
import pytest
import torch

from vllm_ascend_b200 import LLM, SamplingParams
from vllm_ascend_b200.config import ModelConfig
from vllm_ascend_b200.engine import beam

pytestmark = pytest.mark.gpu


def _cfg(dtype="bfloat16"):
    return ModelConfig(name="beams", architecture="Qwen3ForCausalLM", vocab_size=2048, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
                       num_attention_heads=8, num_key_value_heads=2, head_dim=128, qk_norm=True, rope_theta=1e6, dtype=dtype)


def _llm(dtype="bfloat16", **kw):
    return LLM(_cfg(dtype), device="cuda", max_model_len=1024, max_num_seqs=24, max_num_batched_tokens=1024, num_gpu_blocks_override=200,
               block_size=64, cudagraph_capture_sizes=[1, 2, 4, 8, 16, 24], **kw)


def _prompts(*lengths, seed=0):
    rng = np.random.default_rng(seed)
    return [rng.integers(1, 2000, size=n).tolist() for n in lengths]


def _rescored(llm, prompt, tokens):
    """Log-probabilities of an answer's tokens, computed as a prompt."""
    o = llm.generate([prompt + tokens], SamplingParams(temperature=0.0, max_tokens=1, prompt_logprobs=0))
    lps = o[0].prompt_logprobs[len(prompt):]
    return [lp[t] for lp, t in zip(lps, tokens)]


def test_same_beams_as_by_requests_in_32_bits(monkeypatch):
    llm = _llm("float32", enforce_eager=True)
    prompts = _prompts(130, 63, 300)
    ours = llm.beam_search(prompts, beam_width=4, max_tokens=40, ignore_eos=True)
    monkeypatch.setattr(beam, "on_device", lambda *a: False)
    theirs = llm.beam_search(prompts, beam_width=4, max_tokens=40, ignore_eos=True)
    for a, b in zip(ours, theirs):
        assert a[0]["tokens"] == b[0]["tokens"]
        np.testing.assert_allclose([x["cum_logprob"] for x in a], [x["cum_logprob"] for x in b], atol=0.02)


@pytest.mark.parametrize("shared", [False, True])
def test_reported_scores_are_those_of_the_answers(monkeypatch, shared):
    llm = _llm()
    runner = llm.engine.runner
    monkeypatch.setattr(runner, "_sharing_pays", lambda groups: shared)
    prompts = _prompts(200, 129, 64, 700, seed=1)
    found = llm.beam_search(prompts, beam_width=4, max_tokens=24, ignore_eos=True)
    assert any(k[1] == "shared" for k in runner.graphs) == shared            # later rounds replay a graph
    assert runner.stats["graph_replays"] >= 20
    for p, best in zip(prompts, found):
        assert len({tuple(b["tokens"]) for b in best}) == 4
        assert [b["score"] for b in best] == sorted((b["score"] for b in best), reverse=True)
        for b in best[:2]:
            # logits round to bf16: half a step of values up to 8 is 0.016, a token's log-probability takes two; hidden states of prompt and decode
            # kernels differ by roundings of the same size
            assert abs(sum(_rescored(llm, p, b["tokens"])) - b["cum_logprob"]) < 24 * 0.06
    assert not llm.engine.scheduler.requests


def test_hybrid_states_follow_their_beams():
    llm = LLM("tiny-gdn", device="cuda", dtype="float32", max_model_len=256, max_num_seqs=8, num_gpu_blocks_override=64, block_size=16, seed=3, enforce_eager=True)
    rng = np.random.default_rng(2)
    prompts = [rng.integers(1, 500, size=n).tolist() for n in (37, 20)]
    ours = llm.beam_search(prompts, beam_width=3, max_tokens=20, ignore_eos=True)
    for p, best in zip(prompts, ours):
        for b in best:
            assert abs(sum(_rescored(llm, p, b["tokens"])) - b["cum_logprob"]) < 0.02


def test_decode_batches_with_a_common_prefix(monkeypatch):
    rng = np.random.default_rng(5)
    system = rng.integers(1, 2000, size=512).tolist()
    prompts = [system + rng.integers(1, 2000, size=n).tolist() for n in (30, 100, 7, 64, 65, 3)]
    sp = SamplingParams(temperature=0.0, max_tokens=20, ignore_eos=True, logprobs=0)
    outs = []
    for off in (True, False):
        llm = _llm(enable_prefix_caching=True, disable_cascade_attn=off)
        monkeypatch.setattr(llm.engine.runner, "_sharing_pays", lambda groups: True)
        llm.generate([system], SamplingParams(temperature=0.0, max_tokens=1))
        outs.append([o.outputs[0] for o in llm.generate(prompts, sp)])
        assert any(k[1] == "shared" for k in llm.engine.runner.graphs) == (not off)
        torch.cuda.synchronize()
    for a, b in zip(*outs):
        # until roundings choose another token
        n = next((i for i, (x, y) in enumerate(zip(a.token_ids, b.token_ids)) if x != y), len(a.token_ids))
        lp = [[lps[t] for lps, t in zip(o.logprobs, o.token_ids)] for o in (a, b)]
        np.testing.assert_allclose(lp[0][:n], lp[1][:n], atol=0.06)
    assert sum(a.token_ids[:3] == b.token_ids[:3] for a, b in zip(*outs)) >= 4


def test_engines_without_the_kernel_read_every_prefix_for_itself():
    assert _llm().engine.runner.can_share_prefixes()
    assert not _llm("float32", enforce_eager=True, disable_cascade_attn=False).engine.runner.can_share_prefixes()
