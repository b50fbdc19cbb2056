"""Beam search on the engine's own batch: a round is one decode step of all live beams, selection and reordering run on the device.

A prompt is computed once, behind what the prefix cache holds of it.  Its beams are requests that share its full blocks and own a batch row and their partly filled block; the choice of
a round moves what is in those (``ops.reorder_beams``: pages as far as they are filled, recurrent states by batch row), full blocks change hands by
reference.  Attention may read the prompt's keys and values once for all beams (``ops.paged_attention_shared``)."""
from __future__ import annotations

import itertools

import numpy as np
import torch

from .. import _native, ops
from .request import Request, SamplingParams
from .scheduler import Scheduler, SchedulerOutput

_ids = itertools.count()


def _blocks(engine, prompt: int, width: int, max_tokens: int) -> int:
    """Blocks that the beams of a prompt hold at most: the prompt's, and two chains at a time of each beam's own."""
    bs = engine.scheduler.block_size
    return -(-prompt // bs) + 1 + width * (-(-(prompt % bs + max_tokens) // bs) + 1)


def _rows(runner) -> int:
    """Beams that a step holds at most."""
    return min(runner.max_seqs, runner.max_tokens)


def on_device(engine, prompts: list, width: int, max_tokens: int) -> bool:
    """Whether the engine can run these beams itself: one rank that has nothing else to do, no drafts, connectors or adapters, rows and blocks for
    every prompt's beams, as many candidates as the selection takes."""
    r, s, cfg = engine.runner, engine.scheduler, engine.cfg
    par = cfg.parallel
    if type(s) is not Scheduler or engine.has_unfinished() or engine._inflight is not None or r.proposer is not None \
            or engine.kv_connector is not None or engine.eplb is not None or r.lora_manager is not None or r.moe_runtime is not None \
            or r.mm is not None or r.sparse_offload is not None or engine.dp.world_size > 1 or r.pp.world_size > 1 or r.pcp.world_size > 1 \
            or r.dcp_size > 1 or par.tensor_parallel_size > 1:
        return False
    from ..ops.beam import MOST_SELECTED
    return 2 * width <= MOST_SELECTED and width <= _rows(r) and bool(prompts) and all(
        0 < len(p) and len(p) + max_tokens <= s.cfg.max_model_len and _blocks(engine, len(p), width, max_tokens) <= s.pool.num_free_blocks
        for p in prompts)


class _Group:
    """The beams of one prompt: a slot (request) for each, the first ``len(live)`` of them at work."""

    def __init__(self, index: int, prompt: list):
        self.index, self.prompt = index, prompt
        self.slots: list[Request] = []
        self.live: list[tuple] = []                    # (tokens, log-probability), in the order of the slots
        self.done: list[tuple] = []


class BeamSearch:
    def __init__(self, engine, width: int, max_tokens: int, length_penalty: float, ignore_eos: bool):
        self.engine, self.runner, self.scheduler = engine, engine.runner, engine.scheduler
        self.width, self.max_tokens, self.length_penalty = width, max_tokens, length_penalty
        self.eos = None if ignore_eos else engine.eos_token_id
        self.vocab = engine.cfg.model.vocab_size
        self.pages, self.states = self.runner.beam_states()

    def run(self, prompts: list) -> list:
        """``LLM.beam_search`` for as many prompts at a time as rows and blocks allow."""
        results: list = [None] * len(prompts)
        waiting = [_Group(i, p) for i, p in enumerate(prompts)]
        while waiting:
            wave, blocks = [], 0
            while waiting and (len(wave) + 1) * self.width <= _rows(self.runner):
                blocks += _blocks(self.engine, len(waiting[0].prompt), self.width, self.max_tokens)
                if wave and blocks > self.scheduler.pool.num_free_blocks:
                    break
                wave.append(waiting.pop(0))
            try:
                self._wave(wave)
            finally:
                for g in wave:
                    self._release(g)
            for g in wave:
                results[g.index] = self._result(g)
        if self.runner.is_cuda:
            _native.check_status(self.runner.device)
        return results

    # ------------------------------------------------------------------ rounds
    def _wave(self, groups: list) -> None:
        logits = self._prompts(groups)
        scores = torch.zeros((len(groups), 1), dtype=torch.float64, device=logits.device)
        for round_ in range(self.max_tokens):
            k = min(2 * self.width, scores.shape[1] * self.vocab)
            totals, parents, tokens = (t.cpu() for t in ops.beam_select(logits, scores, k, torch.float64))
            chosen = [self._choose(g, *(t[i].tolist() for t in (totals, parents, tokens))) for i, g in enumerate(groups)]
            if round_ + 1 < self.max_tokens:
                going = [(g, p) for g, p in zip(groups, chosen) if p]
                for g in groups:
                    if not g.live:
                        self._release(g)
                self._follow(going)
                groups = [g for g, _ in going]
                if not groups:
                    return
                logits, scores = self._step(groups)

    def _choose(self, g: _Group, totals: list, parents: list, tokens: list) -> list:
        """Takes a group's candidates, best first, until it has its beams; returns the slots that they follow ([]: the group has ended)."""
        nxt, follows = [], []
        for total, p, token in zip(totals, parents, tokens):
            if total == -np.inf:
                break                                  # nothing left that can go on
            beam = (g.live[p][0] + [token], total)
            if token == self.eos:
                g.done.append(beam)
            else:
                nxt.append(beam)
                follows.append(p)
            if len(nxt) >= self.width:
                break
        # a prompt stops once it holds `width` finished beams that beat every live one
        if len(g.done) >= self.width and (not nxt or sorted((self._score(g, b) for b in g.done), reverse=True)[self.width - 1]
                                          >= max(self._score(g, b) for b in nxt)):
            nxt, follows = [], []
        g.live = nxt
        return follows

    def _score(self, g: _Group, beam: tuple) -> float:
        return beam[1] / (max(len(beam[0]) - len(g.prompt), 1) ** self.length_penalty)

    def _result(self, g: _Group) -> list:
        best = sorted(g.done + g.live, key=lambda b: self._score(g, b), reverse=True)[:self.width]
        return [{"tokens": t[len(g.prompt):], "cum_logprob": c, "score": self._score(g, (t, c))} for t, c in best]

    # ------------------------------------------------------------------ steps
    def _prompts(self, groups: list) -> torch.Tensor:
        """Prompts in portions of a step's tokens; logits behind each."""
        budget, kept = self.runner.max_tokens, [None] * len(groups)
        left = []
        for i, g in enumerate(groups):
            req = Request(f"beam-{next(_ids)}", np.asarray(g.prompt, dtype=np.int32), SamplingParams(max_tokens=1, temperature=0.0))
            g.slots, g.live = [req], [(list(g.prompt), 0.0)]
            self.scheduler.reuse(req)
            left.append((i, req))
        while left:
            portions, room = [], budget
            for i, req in left:
                n = min(room, req.num_prompt_tokens - req.num_computed_tokens)
                if n > 0:
                    portions.append((i, req, n))
                    room -= n
            so = self.scheduler.schedule_portions([(req, n) for _, req, n in portions])
            ends, at, by_req = {}, 0, {id(req): i for i, req, _ in portions}
            for req, n in so.scheduled:
                at += n
                if req.num_computed_tokens + n == req.num_prompt_tokens:
                    ends[by_req[id(req)]] = at - 1
            logits = self.runner.device_logits(so, list(ends.values()) or [0])
            for j, i in enumerate(ends):
                kept[i] = logits[j]
            self._computed(so)
            for req, _ in so.scheduled:
                self.scheduler.keep(req)
            left = [(i, req) for i, req in left if i not in ends]
        return torch.stack(kept)

    def _computed(self, so: SchedulerOutput) -> None:
        for req, n in so.scheduled:
            req.num_computed_tokens += n

    def _follow(self, going: list) -> None:
        """Slots take over what their parents have: a first round makes them, later ones exchange."""
        if not going:
            return
        bs, width = self.scheduler.block_size, self.width
        rows = np.full((len(going), width), -1, dtype=np.int32)
        pages, parents, filled = rows.copy(), rows.copy(), np.zeros(len(going), dtype=np.int32)
        for i, (g, follows) in enumerate(going):
            while len(g.slots) < width:
                g.slots.append(self.scheduler.fork(g.slots[0], f"beam-{next(_ids)}"))
            everyone = follows + list(range(len(follows), width))      # slots without a beam stay as they are
            self.scheduler.follow(g.slots, everyone)
            tail = g.slots[0].num_computed_tokens % bs
            filled[i] = tail
            rows[i] = [r.row for r in g.slots]
            parents[i, :len(follows)] = follows
            if tail:
                pages[i] = [r.block_ids[-1] for r in g.slots]
            for r in g.slots:
                n = len(r.block_ids)
                self.runner.block_table_cpu[r.row, :n] = r.block_ids
                self.runner.row_num_blocks[r.row] = n
                self.runner.row_owner[r.row] = r.request_id
        to = lambda x: self.runner._to_dev(torch.from_numpy(x))       # noqa: E731
        parents_on = to(parents)
        if self.pages is not None and filled.any():
            ops.reorder_beams(self.pages, to(pages), parents_on, to(filled))
        if self.states is not None:
            ops.reorder_beams(self.states, to(rows), parents_on)

    def _step(self, groups: list) -> tuple:
        """One token for every live beam; logits and scores of the next selection, groups padded to equal widths."""
        portions = [(g.slots[j], 1) for g in groups for j in range(len(g.live))]
        for g in groups:
            for r, (tokens, _) in zip(g.slots, g.live):
                self.runner.append_tokens(r, tokens[-1:])
        so = self.scheduler.schedule_portions(portions)
        bs = self.scheduler.block_size
        so.shared_groups = [(len(g.live), len(g.prompt) // bs * bs) for g in groups]
        logits = self.runner.device_logits(so)
        self._computed(so)
        for g in groups:                               # slots without a beam keep pace: a later round may need them
            for r in g.slots[len(g.live):]:
                r.num_computed_tokens += 1
                need = self.scheduler._blocks_needed(r, r.num_computed_tokens)
                if need:
                    r.block_ids.extend(self.scheduler.pool.allocate(need))
        wide = max(len(g.live) for g in groups)
        scores = np.full((len(groups), wide), -np.inf, dtype=np.float64)
        index, at = np.zeros((len(groups), wide), dtype=np.int64), 0
        for i, g in enumerate(groups):
            scores[i, :len(g.live)] = [c for _, c in g.live]
            index[i, :len(g.live)] = np.arange(at, at + len(g.live))
            at += len(g.live)
        if at != index.size:
            logits = logits.index_select(0, self.runner._to_dev(torch.from_numpy(index.reshape(-1))))
        return logits, self.runner._to_dev(torch.from_numpy(scores))

    def _release(self, g: _Group) -> None:
        for r in g.slots:
            if r.row >= 0:
                self.runner.row_owner[r.row] = None
            self.scheduler.drop(r)
        g.slots = []
