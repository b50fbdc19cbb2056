"""Host buffers of a step's inputs stay as they are until the step has read them: a device that is late, played on the host."""
import numpy as np
import pytest
import torch
from torch.overrides import TorchFunctionMode

from vllm_ascend_b200 import LLM, SamplingParams


class _LateStream:
    """Asynchronous copies and forward passes run where the host waits for them, in order; steps that sample are waited for."""

    def __init__(self, runner, monkeypatch):
        self.queue, self.mark, self.sampled = [], 0, True
        prepare, forward = runner._prepare_inputs, runner._forward
        stream = self

        class Hold(TorchFunctionMode):
            def __torch_function__(self, func, types, args=(), kwargs=None):
                kwargs = kwargs or {}
                if func is torch.Tensor.copy_ and kwargs.get("non_blocking"):
                    stream.queue.append(lambda to=args[0], what=args[1]: to.copy_(what))
                    return args[0]
                return func(*args, **kwargs)

        def late_prepare(so, pad_to=None):
            with Hold():
                out = prepare(so, pad_to)
            self.sampled = bool(out[3])
            if any(getattr(r, "num_inflight", 0) for r, _ in so.scheduled):      # its last token is put in behind these copies
                self.run(len(self.queue))
            return out

        def late_forward(T, meta):
            out = torch.zeros((T, runner.mcfg.hidden_size), dtype=runner.model.dtype)
            self.queue.append(lambda: out.copy_(forward(T, meta)))
            if self.sampled:
                self.run(len(self.queue))
            return out
        monkeypatch.setattr(runner, "_prepare_inputs", late_prepare)
        monkeypatch.setattr(runner, "_forward", late_forward)
        monkeypatch.setattr(runner, "_inputs_copied", self, raising=False)

    def run(self, n):
        todo, self.queue = self.queue[:n], self.queue[n:]
        for f in todo:
            f()
        self.mark = max(0, self.mark - n)

    def record(self):                                    # as an event's
        self.mark = len(self.queue)

    def synchronize(self):
        self.run(self.mark)


def _llm(**kw):
    return LLM("tiny-qwen", device="cpu", seed=4, block_size=16, max_model_len=256, max_num_seqs=6, max_num_batched_tokens=32, **kw)


def _prompts(*lengths):
    rng = np.random.default_rng(3)
    return [rng.integers(1, 500, size=n).tolist() for n in lengths]


@pytest.mark.parametrize("caching", [False, True])
def test_beams_of_prompts_in_many_portions(monkeypatch, caching):
    want = _llm().beam_search(_prompts(130, 75), beam_width=3, max_tokens=5, ignore_eos=True)
    llm = _llm(enable_prefix_caching=caching)
    _LateStream(llm.engine.runner, monkeypatch)
    for _ in range(2):                                   # a second time from the prefix cache
        got = llm.beam_search(_prompts(130, 75), beam_width=3, max_tokens=5, ignore_eos=True)
        assert [[b["tokens"] for b in best] for best in got] == [[b["tokens"] for b in best] for best in want]


@pytest.mark.parametrize("asynchronous", [False, True])
def test_prompts_in_many_portions(monkeypatch, asynchronous):
    sp = SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True)
    want = [o.outputs[0].token_ids for o in _llm(async_scheduling=asynchronous).generate(_prompts(130, 75), sp)]
    llm = _llm(async_scheduling=asynchronous)
    _LateStream(llm.engine.runner, monkeypatch)
    assert [o.outputs[0].token_ids for o in llm.generate(_prompts(130, 75), sp)] == want
