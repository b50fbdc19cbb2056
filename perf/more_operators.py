"""Beam search on the device, as the workloads its operators are timed on.

A step of a beam search over ``groups`` prompts with ``width`` beams each has logits for every beam and does three things:

  select    the best continuations of every group: a beam's score so far plus the log-probability of a token, over all beams and
            the whole vocabulary of a group, best first, ties to the lowest beam and token.  Beams that ended have the score
            -inf; rows without a distribution (a NaN, +inf or nothing finite among the logits) have no candidates
  reorder   the beams' states follow the chosen parents, in place and for all layers at once: rows of recurrent states, or the
            pages that beams have of their own, as far as they are filled
  attention the next step's tokens over prompts that the beams of a group share: the keys and values in front of ``prefix`` lie in
            the same pages for all sequences of a group, what follows in pages of their own.  The same batches come from requests
            behind one system prompt, or several questions about one document

Sizes are ragged and odd around what a case names, pages lie scattered in their caches.
"""
from __future__ import annotations

import math
import random
import zlib

import torch

own = False

HEADS = [(32, 8), (32, 8), (64, 8), (32, 4), (16, 4), (28, 4), (16, 16), (8, 1), (6, 2)]


def _select(name, groups, width, vocab, dtype="bf16", masked=0.0, ended=0.0):
    return {"name": name, "op": "select", "groups": groups, "width": width, "vocab": vocab, "dtype": dtype, "masked": masked,
            "ended": ended}


def _reorder(name, kind, groups, width, layers, heads, dim, page=0):
    return {"name": name, "op": "reorder", "kind": kind, "groups": groups, "width": width, "layers": layers, "heads": heads,
            "dim": dim, "page": page}


def _attend(name, heads, dim, page, groups, width, prefix, tail, each=1):
    return {"name": name, "op": "attention", "heads": heads[0], "kv_heads": heads[1], "dim": dim, "page": page, "groups": groups,
            "width": width, "prefix": prefix, "tail": tail, "each": each}


def listed():
    return [
        _select("select 1x4 of 32000", 1, 4, 32000, "fp32"),                     # one user, four beams: latency
        _select("select 8x8 of 151936", 8, 8, 151936),                           # a usual batch of translations
        _select("select 5x3 of 50001, masked", 5, 3, 50001, "fp32", 0.9, 0.2),   # guided answers, ended beams, odd rows
        _select("select 96x8 of 151936", 96, 8, 151936, ended=0.05),             # an offline batch
        _reorder("reorder pages 1x4", "pages", 1, 4, 36, 8, 128, 128),           # one user: latency, all layers of a model
        _reorder("reorder pages 16x8", "pages", 16, 8, 12, 8, 128, 64),          # an offline batch
        _reorder("reorder states 16x4", "states", 16, 4, 4, 32, 128),            # recurrent states, convolution windows
        _attend("attention 1x4 over 1500", (32, 8), 128, 128, 1, 4, 1536, 40),   # one user, four beams: latency
        _attend("attention 16x8 over 2000", (32, 8), 128, 128, 16, 8, 2048, 100),            # an offline batch of beams
        _attend("attention 1x8 over 60000", (64, 8), 128, 128, 1, 8, 60000, 300),            # questions about one long document
        _attend("attention 1x192 over 2000", (32, 8), 128, 128, 1, 192, 2048, 900),          # requests behind one system prompt
        _attend("attention 9x4x4 over 5000", (28, 4), 64, 16, 9, 4, 5000, 700, each=4),      # drafts to verify, small heads
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["select", "reorder", "attention", "attention"])
    if op == "select":
        vocab, width = _log(rng, 500, 256000), _log(rng, 1, 64)
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        most = 115_000_000 // (2 if dtype == "fp32" else 1)
        c = _select("", _log(rng, 1, max(1, min(256, most // (width * vocab)))), width, vocab, dtype,
                    rng.choice([0.0, 0.0, 0.5, 0.99]), rng.choice([0.0, 0.0, 0.3]))
    elif op == "reorder":
        width = _log(rng, 1, 64)
        kind = rng.choice(["pages", "pages", "states"])
        heads, dim = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128])
        page = rng.choice([16, 32, 64, 128]) if kind == "pages" else 0
        layers = _log(rng, 1, 48)
        row = heads * dim * (page * 4 if page else dim * 4)                      # bytes of a beam in a layer
        c = _reorder("", kind, _log(rng, 1, max(1, min(128, 400_000_000 // (row * layers * width)))), width, layers, heads, dim, page)
        c["layers"] = max(1, min(layers, 400_000_000 // (row * c["groups"] * width)))
    else:
        heads, dim, page = rng.choice(HEADS), rng.choice([128, 128, 64]), rng.choice([16, 32, 64, 128, 128])
        each = rng.choice([1, 1, 1, 2, 4])
        c = _attend("", heads, dim, page, _log(rng, 1, 32), 0, 0, 0, each)
        c["width"] = _log(rng, 1, max(1, 192 // c["groups"]))
        seqs = c["groups"] * c["width"]
        most = min(40000, 600_000 // (c["groups"] * heads[1]), 3_000_000_000 // (seqs * each * heads[0] * dim))
        c["prefix"] = _log(rng, page, max(page + 1, most))
        c["tail"] = _log(rng, 1, max(2, min(4000, 600_000 // (seqs * heads[1]))))
    del c["name"]
    return c


# ---------------------------------------------------------------- what a case holds
def _gen(*what):
    g = torch.Generator(device="cuda")
    g.manual_seed(zlib.crc32(repr(what).encode()))
    return g


def _plain(c):
    return sorted((k, v) for k, v in c.items() if k != "name")


def _around(rng, x, n):
    return [max(1, round(x * rng.uniform(0.6, 1.4))) if n > 1 else max(1, x) for _ in range(n)]


def _parents(c):
    """(parent of every beam, filled tokens of its page) per group: good beams have several children."""
    rng = random.Random(repr(_plain(c)))
    parents = []
    for _ in range(c["groups"]):
        best = [rng.expovariate(1.0) for _ in range(c["width"])]
        parents.append(rng.choices(range(c["width"]), weights=best, k=c["width"]))
    return parents, [rng.randint(1, c["page"]) if c["page"] else 0 for _ in range(c["groups"])]


def _lengths(c):
    """Of every group its sequences and the length of its prefix; of every sequence the tokens behind the prefix, new ones included."""
    rng = random.Random(repr(_plain(c)))
    width = _around(rng, c["width"], c["groups"])
    prefix = [max(1, n // c["page"]) * c["page"] for n in _around(rng, c["prefix"], c["groups"])]
    return width, prefix, [n + c["each"] for n in _around(rng, c["tail"], sum(width))]


def _select_inputs(c, seed):
    g = _gen(seed, _plain(c))
    rows, v = c["groups"] * c["width"], c["vocab"]
    logits = torch.empty((rows, v), dtype=torch.float32, device="cuda").normal_(std=2.2, generator=g)
    sure = torch.randint(0, v, (rows, 6), generator=g, device="cuda")            # the words that a row is about
    logits.scatter_add_(1, sure, torch.empty((rows, 6), device="cuda").uniform_(4.0, 11.0, generator=g))
    if c["masked"]:
        logits.masked_fill_(torch.empty((rows, v), device="cuda").uniform_(generator=g) < c["masked"], -math.inf)
    scores = -torch.empty((c["groups"], c["width"]), device="cuda").exponential_(generator=g) * 5 - 3
    if c["ended"]:
        scores.masked_fill_(torch.empty(scores.shape, device="cuda").uniform_(generator=g) < c["ended"], -math.inf)
    return {"logits": logits.bfloat16() if c["dtype"] == "bf16" else logits, "scores": scores, "k": min(2 * c["width"], v)}


def _reorder_inputs(c, seed):
    g = _gen(seed, _plain(c))
    n, w = c["groups"], c["width"]
    held = n * w + 3                                                             # other rows and pages stay as they are
    if c["kind"] == "pages":                                                     # [pages, tokens, heads, channels], a head's page in one run
        shapes = [((2 * c["layers"], held, c["heads"], c["page"], c["dim"]), torch.bfloat16)]
    else:                                                                        # windows of convolutions, recurrent states
        shapes = [((c["layers"], held, 3 * c["heads"] * c["dim"], 3), torch.bfloat16),
                  ((c["layers"], held, c["heads"], c["dim"], c["dim"]), torch.float32)]
    memory = [torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g) for shape, dtype in shapes]
    if c["kind"] == "pages":
        memory = [m.transpose(2, 3) for m in memory]
    rows = torch.randperm(held, generator=g, device="cuda")[:n * w].int().view(n, w)
    parents, filled = _parents(c)
    return {"memory": memory, "tensors": [t for m in memory for t in m], "rows": rows,
            "parents": torch.tensor(parents, dtype=torch.int32, device="cuda"),
            "filled": torch.tensor(filled, dtype=torch.int32, device="cuda") if c["page"] else None}


def _attend_inputs(c, seed):
    g = _gen(seed, _plain(c))
    width, prefix, tail = _lengths(c)
    page, hkv, d = c["page"], c["kv_heads"], c["dim"]
    first = [0]
    for n in width:
        first.append(first[-1] + n)
    shared = [n // page for n in prefix]
    behind = [-(-n // page) for n in tail]
    blocks = sum(shared) + sum(behind) + 3
    ids = torch.randperm(blocks, generator=g, device="cuda").int()
    lens, at = [], 0
    group_of = [i for i, n in enumerate(width) for _ in range(n)]
    table = torch.zeros((first[-1], max(shared[group_of[s]] + behind[s] for s in range(first[-1]))), dtype=torch.int32, device="cuda")
    for i, n in enumerate(shared):
        table[first[i]:first[i + 1], :n] = ids[at:at + n]
        at += n
    for s, n in enumerate(behind):
        table[s, shared[group_of[s]]:shared[group_of[s]] + n] = ids[at:at + n]
        at += n
        lens.append(prefix[group_of[s]] + tail[s])
    caches = []
    for scale in (1.0, 0.3):
        t = torch.empty((blocks, hkv, page, d), dtype=torch.bfloat16, device="cuda").normal_(std=scale, generator=g)
        caches.append(t.transpose(1, 2))
    caches[0][..., torch.randperm(d, generator=g, device="cuda")[:d // 16]] *= 4.0      # channels above the others, as trained keys have
    rows = torch.empty((first[-1] * c["each"], c["heads"] + 2 * hkv, d), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    return {"q": rows[:, :c["heads"]], "k": caches[0], "v": caches[1], "table": table, "lens": lens, "first": first, "prefix": prefix,
            "scale": 0.7 * d ** -0.5}


def prepare(case, seed):
    c = case
    if c["op"] == "select":
        return dict(_select_inputs(c, seed), case=c)
    if c["op"] == "reorder":
        state = dict(_reorder_inputs(c, seed), case=c)
        if own:
            from vllm_ascend_b200 import ops
            state["handle"] = ops.beam_states(state["tensors"], paged=c["kind"] == "pages")      # kept as long as the caches live
        return state
    state = dict(_attend_inputs(c, seed), case=c)
    if own:
        from vllm_ascend_b200 import ops
        from vllm_ascend_b200.attention.metadata import metadata_from_tensors
        new, lens = c["each"], state["lens"]
        starts = torch.arange(0, (len(lens) + 1) * new, new, device="cuda").int()
        state["meta"] = metadata_from_tensors(starts, torch.tensor(lens, dtype=torch.int32, device="cuda"), state["table"], new, max(lens),
                                              c["heads"], c["kv_heads"], c["dim"])
        # made once a step, for all layers
        state["plan"] = ops.plan_shared_prefix(state["meta"], torch.tensor(state["first"], dtype=torch.int32, device="cuda"),
                                               torch.tensor(state["prefix"], dtype=torch.int32, device="cuda"), c["heads"], c["kv_heads"])
    return state


# ---------------------------------------------------------------- plain forms
def _select_plain(state):
    scores, k = state["scores"], state["k"]
    n, w = scores.shape
    x = state["logits"].double()                       # candidates next to one another are told apart in 64 bits
    top = x.amax(-1, keepdim=True)
    total = scores.double().reshape(-1, 1) + (x - top - (x - top).exp().sum(-1, keepdim=True).log())
    total = total.nan_to_num_(nan=-math.inf, posinf=-math.inf, neginf=-math.inf).view(n, -1)
    places = torch.arange(total.shape[1], device=x.device)
    taken = torch.zeros_like(total, dtype=torch.bool)
    values, found = [], []
    for _ in range(k):
        best = total.amax(-1)
        at = torch.where((total == best[:, None]) & ~taken, places, total.shape[1]).amin(-1)
        values.append(best)
        found.append(at)
        taken.scatter_(1, at[:, None], True)
        total.scatter_(1, at[:, None], -math.inf)
    at = torch.stack(found, 1)
    v = x.shape[1]
    return torch.stack(values, 1).float(), (at // v).int(), at % v


def _reorder_plain(state):
    rows, filled = state["rows"].long(), state["filled"]
    n, w = rows.shape
    to = rows.reshape(-1)
    source = rows.gather(1, state["parents"].long()).reshape(-1)
    for t in state["tensors"]:
        old = t[source]
        if filled is not None:
            mine = torch.arange(t.shape[1], device=t.device) < filled.repeat_interleave(w)[:, None]
            old = torch.where(mine[:, :, None, None], old, t[to])
        t[to] = old
    return state["memory"]


def _attend_plain(state):
    c, q, page = state["case"], state["q"], state["case"]["page"]
    group, new = c["heads"] // c["kv_heads"], c["each"]
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    for i, prefix in enumerate(state["prefix"]):
        k0 = v0 = None
        for s in range(state["first"][i], state["first"][i + 1]):
            n = state["lens"][s]

            def rows(cache, lo, hi):
                pos = torch.arange(lo, hi, device=q.device)
                return cache[state["table"][s][pos // page].long(), pos % page].float().transpose(0, 1)       # [heads, keys, channels]
            if k0 is None:
                k0, v0 = rows(state["k"], 0, prefix), rows(state["v"], 0, prefix)
            k1, v1 = rows(state["k"], prefix, n), rows(state["v"], prefix, n)
            rows_q = q[s * new:(s + 1) * new].float().transpose(0, 1).reshape(c["kv_heads"], group * new, c["dim"])
            a, b = (rows_q @ k.transpose(1, 2) * state["scale"] for k in (k0, k1))
            mine = torch.arange(n - new, n, device=q.device).repeat(group)[:, None]
            b = b.masked_fill(torch.arange(prefix, n, device=q.device) > mine, -math.inf)
            top = torch.maximum(a.amax(-1, keepdim=True), b.amax(-1, keepdim=True))
            a, b = (a - top).exp(), (b - top).exp()
            o = (a @ v0 + b @ v1) / (a.sum(-1, keepdim=True) + b.sum(-1, keepdim=True))
            out[s * new:(s + 1) * new] = o.view(c["heads"], new, c["dim"]).transpose(0, 1).to(q.dtype)
    return out


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"select": _select_plain, "reorder": _reorder_plain, "attention": _attend_plain}[op](state)
    from vllm_ascend_b200 import ops
    if op == "select":
        return ops.beam_select(state["logits"], state["scores"], state["k"])
    if op == "reorder":
        ops.reorder_beams(state["handle"], state["rows"], state["parents"], state["filled"])
        return state["memory"]
    return ops.paged_attention_shared(state["q"], state["k"], state["v"], state["meta"], state["plan"], state["scale"])


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "select":
        elements = c["groups"] * c["width"] * c["vocab"]
        return {"bytes": elements * (2 if c["dtype"] == "bf16" else 4) + c["groups"] * c["width"] * 36, "flops": 4 * elements}
    if c["op"] == "reorder":
        moved = 0
        for parents, filled in zip(*_parents(c)):
            change = [w for w, p in enumerate(parents) if p != w]
            rows = len(change) + len({parents[w] for w in change})               # written and read
            if c["kind"] == "pages":
                moved += rows * c["layers"] * 2 * filled * c["heads"] * c["dim"] * 2
            else:
                moved += rows * c["layers"] * c["heads"] * c["dim"] * (9 * 2 + c["dim"] * 4)
        return {"bytes": moved, "flops": 0}
    width, prefix, tail = _lengths(c)
    token = c["kv_heads"] * c["dim"] * 2 * 2                                     # bytes of a token's keys and values
    nbytes = (sum(prefix) + sum(tail)) * token + 2 * sum(width) * c["each"] * c["heads"] * c["dim"] * 2
    new = c["each"]
    pairs = sum(n * p for n, p in zip(width, prefix)) * new + sum(new * n - new * (new - 1) // 2 for n in tail)
    return {"bytes": nbytes, "flops": 4 * pairs * c["heads"] * c["dim"]}


# ---------------------------------------------------------------- in 64 bits, from the definition
def exact(case, seed):
    c = case
    if c["op"] == "select":
        x = _select_inputs(c, seed)
        logits, scores = x["logits"], x["scores"]
        v, outs = c["vocab"], []
        for g in range(c["groups"]):
            lp = torch.log_softmax(logits[g * c["width"]:(g + 1) * c["width"]].double(), -1) + scores[g].double()[:, None]
            lp = torch.where(lp.isfinite(), lp, -math.inf).reshape(-1)
            best, at = torch.sort(lp, descending=True, stable=True)
            outs.append((best[:x["k"]].clone(), (at[:x["k"]] // v).int(), at[:x["k"]] % v))
        return tuple(torch.stack(part) for part in zip(*outs))
    if c["op"] == "reorder":
        x = _reorder_inputs(c, seed)
        parents, filled = _parents(c)
        rows = x["rows"].tolist()
        for t in x["tensors"]:
            before = t.clone()
            for g, (mine, from_) in enumerate(zip(rows, parents)):
                for w, p in enumerate(from_):
                    if c["page"]:
                        t[mine[w], :filled[g]] = before[mine[p], :filled[g]]
                    else:
                        t[mine[w]] = before[mine[p]]
        return x["memory"]
    x = _attend_inputs(c, seed)
    q, new, per = x["q"].double(), c["each"], c["heads"] // c["kv_heads"]
    outs = []
    for s, n in enumerate(x["lens"]):
        keys = torch.arange(n, device=q.device)
        at, off = x["table"][s].long()[keys // c["page"]], keys % c["page"]
        seen = keys[None] <= torch.arange(n - new, n, device=q.device)[:, None]
        rows = q[s * new:(s + 1) * new].unflatten(1, (c["kv_heads"], per))
        p = torch.einsum("tghd,kgd->ghtk", rows, x["k"][at, off].double()) * x["scale"]
        p = torch.softmax(torch.where(seen, p, -math.inf), -1)
        outs.append(torch.einsum("ghtk,kgd->tghd", p, x["v"][at, off].double()).flatten(1, 2))
    return torch.cat(outs)
