"""Steps that would share prefixes replay the graph that is there until theirs is captured."""
import numpy as np
import pytest
import torch

from vllm_ascend_b200 import LLM
from vllm_ascend_b200.compilation.cuda_graph import BatchDescriptor
from vllm_ascend_b200.engine.request import Request, SamplingParams


class _Graphs:
    def __init__(self, hidden):
        self.hidden, self.log, self.entries = hidden, [], {}

    def capture(self, desc, tokens, meta):
        self.log.append(("capture", desc))

    def replay(self, desc):
        self.log.append(desc)
        return self.hidden


@pytest.fixture
def engine(monkeypatch):
    llm = LLM("tiny-qwen", device="cpu", seed=1, block_size=16, max_model_len=128, max_num_seqs=8)
    runner = llm.engine.runner
    graphs = _Graphs(torch.zeros(4, runner.mcfg.hidden_size))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    runner.capture_sizes, runner.graph_wrapper = [4], graphs
    runner.graphs[(4, False)] = BatchDescriptor(num_tokens=4)
    return llm.engine, graphs


def _beams(engine, n):
    s, reqs = engine.scheduler, []
    for i in range(n):
        r = Request(f"r{i}", np.arange(1, 34, dtype=np.int32), SamplingParams(max_tokens=1))
        s.schedule_portions([(r, 33)])
        r.num_computed_tokens = 32
        reqs.append(r)
    return reqs


def test_the_plain_graph_serves_until_the_shared_one_is_captured(engine):
    engine, graphs = engine
    reqs, runner = _beams(engine, 3), engine.runner
    plain = runner.graphs[(4, False)]
    for _ in range(4):
        so = engine.scheduler.schedule_portions([(r, 1) for r in reqs])
        so.shared_groups = [(3, 32)]
        runner.device_logits(so)
    shared = BatchDescriptor(num_tokens=4, shared_prefixes=True)
    assert graphs.log == [plain, plain, ("capture", shared), shared, shared]
    assert runner.stats["graph_replays"] == 4 and runner.stats["eager_steps"] == 0


def test_sizes_without_a_graph_share_eagerly(engine, monkeypatch):
    engine, graphs = engine
    from vllm_ascend_b200 import ops
    reqs, runner, calls = _beams(engine, 5), engine.runner, []
    plan = ops.plan_shared_prefix
    monkeypatch.setattr(ops, "plan_shared_prefix", lambda *a: calls.append(1) or plan(*a))
    so = engine.scheduler.schedule_portions([(r, 1) for r in reqs])
    so.shared_groups = [(5, 32)]
    runner.device_logits(so)
    assert calls and not graphs.log and runner.stats["eager_steps"] == 1
