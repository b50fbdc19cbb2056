"""Beam search on the engine's own batch against beam search by requests, on the host."""
import numpy as np
import pytest

from vllm_ascend_b200 import LLM
from vllm_ascend_b200.engine import beam


def _prompts(*lengths, seed=0, vocab=500):
    rng = np.random.default_rng(seed)
    return [rng.integers(1, vocab, size=n).tolist() for n in lengths]


def _both(llm, monkeypatch, prompts, **kw):
    calls = []
    run = beam.BeamSearch.run
    monkeypatch.setattr(beam.BeamSearch, "run", lambda self, p: calls.append(1) or run(self, p))
    ours = llm.beam_search(prompts, **kw)
    assert calls                                        # on the engine's own batch
    monkeypatch.setattr(beam, "on_device", lambda *a: False)
    theirs = llm.beam_search(prompts, **kw)
    monkeypatch.undo()
    return ours, theirs


def _same(ours, theirs):
    assert len(ours) == len(theirs)
    for a, b in zip(ours, theirs):
        assert [x["tokens"] for x in a] == [x["tokens"] for x in b]
        np.testing.assert_allclose([x["score"] for x in a], [x["score"] for x in b], atol=2e-4)


def _idle(llm, blocks):
    s = llm.engine.scheduler
    assert not s.requests and not s.running and len(s._free_rows) == s.cfg.max_num_seqs and s.pool.num_free_blocks == blocks


@pytest.mark.parametrize("width,tokens,lengths", [(1, 6, (9,)), (3, 9, (11, 7, 30)), (4, 20, (16, 32, 5)), (2, 35, (17,))])
def test_same_beams_as_by_requests(monkeypatch, width, tokens, lengths):
    llm = LLM("tiny-qwen", device="cpu", seed=1, block_size=16, max_model_len=128, max_num_seqs=16)
    free = llm.engine.scheduler.pool.num_free_blocks
    _same(*_both(llm, monkeypatch, _prompts(*lengths), beam_width=width, max_tokens=tokens, ignore_eos=True, length_penalty=0.8))
    _idle(llm, free)


def test_beams_that_end(monkeypatch):
    llm = LLM("tiny-qwen", device="cpu", seed=2, block_size=16, max_model_len=128, max_num_seqs=12)
    free = llm.engine.scheduler.pool.num_free_blocks
    prompts = _prompts(11, 20, 6, seed=3)
    plain = llm.beam_search(prompts, beam_width=3, max_tokens=8, ignore_eos=True)
    for eos in {b["tokens"][i] for best in plain for b in best[:2] for i in (1, 3)}:
        llm.engine.eos_token_id = eos
        _same(*_both(llm, monkeypatch, prompts, beam_width=3, max_tokens=8))
        _idle(llm, free)


def test_more_prompts_than_rows_and_prompts_longer_than_a_step(monkeypatch):
    llm = LLM("tiny-qwen", device="cpu", seed=4, block_size=16, max_model_len=128, max_num_seqs=5, max_num_batched_tokens=24)
    free = llm.engine.scheduler.pool.num_free_blocks
    _same(*_both(llm, monkeypatch, _prompts(40, 12, 70, 24, 25, seed=5), beam_width=2, max_tokens=5, ignore_eos=True))
    _idle(llm, free)


def test_few_blocks(monkeypatch):
    llm = LLM("tiny-qwen", device="cpu", seed=4, block_size=16, max_model_len=96, max_num_seqs=8, num_gpu_blocks_override=22)
    free = llm.engine.scheduler.pool.num_free_blocks
    _same(*_both(llm, monkeypatch, _prompts(40, 33, 20, seed=6), beam_width=3, max_tokens=20, ignore_eos=True))
    _idle(llm, free)


def test_shared_prefixes_are_used_and_change_nothing(monkeypatch):
    from vllm_ascend_b200 import ops
    llm = LLM("tiny-qwen", device="cpu", seed=1, block_size=16, max_model_len=128, max_num_seqs=16)
    calls = []
    shared = ops.paged_attention_shared
    monkeypatch.setattr(ops, "paged_attention_shared", lambda *a, **k: calls.append(a[4].prefix_lens.tolist()) or shared(*a, **k))
    with_plan = llm.beam_search(_prompts(33, 20), beam_width=3, max_tokens=5, ignore_eos=True)
    assert calls and calls[0][:2] == [32, 16]
    monkeypatch.setattr(llm.engine.runner, "can_share_prefixes", lambda: False)
    calls.clear()
    _same(with_plan, llm.beam_search(_prompts(33, 20), beam_width=3, max_tokens=5, ignore_eos=True))
    assert not calls


def test_decode_batches_with_a_common_prefix():
    from vllm_ascend_b200 import SamplingParams, ops
    rng = np.random.default_rng(7)
    system = rng.integers(1, 500, size=40).tolist()
    prompts = [system + rng.integers(1, 500, size=n).tolist() for n in (3, 9, 5)]
    sp = SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True)
    outs, calls = [], []
    shared = ops.paged_attention_shared
    for off in (True, False):
        llm = LLM("tiny-qwen", device="cpu", seed=1, block_size=16, max_model_len=128, max_num_seqs=8, enable_prefix_caching=True,
                  disable_cascade_attn=off)
        llm.generate([system], SamplingParams(temperature=0.0, max_tokens=1))
        try:
            ops.paged_attention_shared = lambda *a, **k: calls.append(a[4].prefix_lens.tolist()) or shared(*a, **k)
            outs.append([o.outputs[0].token_ids for o in llm.generate(prompts, sp)])
        finally:
            ops.paged_attention_shared = shared
        assert bool(calls) == (not off)
    assert outs[0] == outs[1] and any(c[0] == 32 for c in calls)


@pytest.mark.parametrize("model,extra", [("tiny-gdn", {}), ("tiny-deepseek-sparse", {"index_topk": 96}), ("tiny-pegopel", {}), ("tiny-dubizen", {}), ("tiny-moe", {}),
                                         ("tiny-nevotar", {}), ("tiny-vofelix", {})])
def test_other_kinds_of_layers(monkeypatch, model, extra):
    from vllm_ascend_b200.config import get_model_config
    # (sparse attention that selects all keys: which it selects beyond that follows the last bit of a score)
    llm = LLM(get_model_config(model, **extra), device="cpu", seed=3, block_size=16, max_model_len=96, max_num_seqs=8)
    free = llm.engine.scheduler.pool.num_free_blocks
    ours, theirs = _both(llm, monkeypatch, _prompts(21, 9, seed=8, vocab=120), beam_width=3, max_tokens=14, ignore_eos=True)
    _same(ours, theirs)
    _idle(llm, free)


def test_a_cache_of_four_bits(monkeypatch):
    from vllm_ascend_b200.config import get_model_config
    cfg = get_model_config("tiny-qwen")
    cfg.head_dim = 64
    llm = LLM(cfg, device="cpu", seed=3, block_size=16, max_model_len=96, max_num_seqs=8, kv_cache_dtype="int4")
    # by requests every round computes whole sequences again, from rows that were never rounded: other beams may come out ahead
    ours, theirs = _both(llm, monkeypatch, _prompts(21, 9, seed=8), beam_width=2, max_tokens=18, ignore_eos=True)
    for a, b in zip(ours, theirs):
        assert abs(a[0]["score"] - b[0]["score"]) < 0.5 and len(a) == len(b) == 2


def test_engines_that_search_by_requests(monkeypatch):
    llm = LLM("tiny-qwen", device="cpu", seed=1, block_size=16, max_model_len=64, max_num_seqs=4)
    monkeypatch.setattr(beam.BeamSearch, "run", lambda self, p: pytest.fail("not this engine's"))
    assert not beam.on_device(llm.engine, [[1] * 10], 5, 4)                 # more beams than rows
    assert not beam.on_device(llm.engine, [[1] * 60], 2, 10)                # past the model's length
    assert not beam.on_device(llm.engine, [], 2, 4)
    llm.engine.runner.lora_manager = object()
    assert not beam.on_device(llm.engine, [[1] * 10], 2, 4)
    llm.engine.runner.lora_manager = None
    assert beam.on_device(llm.engine, [[1] * 10], 2, 4)
    assert llm.beam_search([], beam_width=2, max_tokens=3) == []


def test_prompts_begin_behind_what_the_prefix_cache_holds(monkeypatch):
    llm = LLM("tiny-qwen", device="cpu", seed=1, block_size=16, max_model_len=128, max_num_seqs=16, enable_prefix_caching=True)
    free = llm.engine.scheduler.pool.num_free_blocks
    steps = []
    runner = llm.engine.runner
    logits = runner.device_logits
    monkeypatch.setattr(runner, "device_logits", lambda so, rows=None: steps.append(so.num_scheduled_tokens) or logits(so, rows))
    prompts = _prompts(33, 64, 40)
    first = llm.beam_search(prompts, beam_width=3, max_tokens=20, ignore_eos=True)
    assert steps[0] == 33 + 64 + 40
    _idle(llm, free)
    steps.clear()
    _same(llm.beam_search(prompts, beam_width=3, max_tokens=20, ignore_eos=True), first)
    assert steps[0] == 1 + 16 + 8                        # a last token is always computed
    steps.clear()
    _same(llm.beam_search([p + [7] for p in prompts], beam_width=2, max_tokens=3, ignore_eos=True),
          LLM("tiny-qwen", device="cpu", seed=1, block_size=16, max_model_len=128, max_num_seqs=16).beam_search(
              [p + [7] for p in prompts], beam_width=2, max_tokens=3, ignore_eos=True))
    assert steps[0] == 2 + 1 + 9
    _idle(llm, free)


def test_engines_that_read_every_prefix_for_itself():
    assert LLM("tiny-qwen", device="cpu", max_model_len=64, max_num_seqs=2).engine.runner.can_share_prefixes()
    for model, kw in (("tiny-qwen", {"speculative_config": {"method": "ngram", "num_speculative_tokens": 2}}), ("tiny-qwen", {"kv_cache_dtype": "int4"}),
                      ("tiny-gdn", {})):
        from vllm_ascend_b200.config import get_model_config
        cfg = get_model_config(model)
        if kw.get("kv_cache_dtype"):
            cfg.head_dim = 64
        assert not LLM(cfg, device="cpu", max_model_len=64, max_num_seqs=2, disable_cascade_attn=False, **kw).engine.runner.can_share_prefixes()


def test_steps_keep_within_their_tokens(monkeypatch):
    llm = LLM("tiny-qwen", device="cpu", seed=1, block_size=16, max_model_len=128, max_num_seqs=16, max_num_batched_tokens=8)
    logits, steps = llm.engine.runner.device_logits, []
    monkeypatch.setattr(llm.engine.runner, "device_logits", lambda so, rows=None: steps.append(so.num_scheduled_tokens) or logits(so, rows))
    prompts = _prompts(11, 7, 30)
    found = llm.beam_search(prompts, beam_width=4, max_tokens=5, ignore_eos=True)
    assert steps and max(steps) <= 8
    _same(found, LLM("tiny-qwen", device="cpu", seed=1, block_size=16, max_model_len=128, max_num_seqs=16).beam_search(
        prompts, beam_width=4, max_tokens=5, ignore_eos=True))
    assert not beam.on_device(llm.engine, prompts, 9, 5)
