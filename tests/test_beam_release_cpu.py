"""A beam search that ends with an error leaves no block, row or entry behind."""
import numpy as np
import pytest

from vllm_ascend_b200 import LLM


def _prompts(*lengths):
    rng = np.random.default_rng(3)
    return [rng.integers(1, 500, size=n).tolist() for n in lengths]


@pytest.mark.parametrize("step", [0, 1, 3, 5])
def test_an_error_in_any_step(monkeypatch, step):
    llm = LLM("tiny-qwen", device="cpu", seed=1, block_size=16, max_model_len=128, max_num_seqs=8, max_num_batched_tokens=40, enable_prefix_caching=True)
    s, prompts = llm.engine.scheduler, _prompts(50, 33, 20, 64)
    free = s.pool.num_free_blocks
    want = llm.beam_search(prompts, beam_width=2, max_tokens=4, ignore_eos=True)      # the prompts are in the prefix cache now
    logits, steps = llm.engine.runner.device_logits, []

    def fails(so, rows=None):
        steps.append(1)
        if len(steps) > step:
            raise RuntimeError("out of memory")
        return logits(so, rows)
    monkeypatch.setattr(llm.engine.runner, "device_logits", fails)
    with pytest.raises(RuntimeError, match="out of memory"):
        llm.beam_search([p + [1] * 41 for p in prompts], beam_width=2, max_tokens=4, ignore_eos=True)
    assert s.pool.num_free_blocks == free and not s._hashes and not s.requests and not s.running and len(s._free_rows) == 8
    monkeypatch.undo()
    assert llm.beam_search(prompts, beam_width=2, max_tokens=4, ignore_eos=True)[0][0]["tokens"] == want[0][0]["tokens"]
