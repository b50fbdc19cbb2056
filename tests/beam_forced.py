"""Beam searches that take given choices, and the logits of their rounds."""
import torch

from vllm_ascend_b200 import ops


def sharpen(llm, factor=2.0):
    """Larger queries: attention to few keys, so that a key missing or of another sequence shows."""
    for layer in llm.engine.runner.model.layers:
        layer.self_attn.q_norm.mul_(factor)
    return llm


def search(llm, monkeypatch, prompts, width, rounds, share, choices=None):
    """(logits of every round's beams, choices of every round); ``choices``: taken instead of the search's own."""
    seen, taken = [], []
    select = ops.beam_select

    def record(logits, scores, *args):
        seen.append(logits.float().cpu()[scores.reshape(-1).isfinite().cpu()])
        out = select(logits, scores, *args) if choices is None else tuple(t.to(logits.device) for t in choices[len(taken)])
        taken.append(tuple(t.cpu().clone() for t in out))
        return out
    with monkeypatch.context() as m:
        m.setattr(ops, "beam_select", record)
        m.setattr(llm.engine.runner, "_sharing_pays", lambda groups: share)
        llm.beam_search(prompts, beam_width=width, max_tokens=rounds, ignore_eos=True)
    return seen, taken


def worst(a, b, slack):
    """The largest difference of two searches' logits in units of ``slack(row)``."""
    assert len(a) == len(b) and all(x.shape == y.shape for x, y in zip(a, b))
    return max(float(((x - y).abs().amax(-1) / torch.stack([slack(r) for r in x])).max()) for x, y in zip(a, b))
