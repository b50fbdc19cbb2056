"""The cache of keys and values in 4 bits, as the workloads its operators are timed on.

Groups of 32 adjacent channels of a token and head share a scale s, the smallest number of five significant bits with 7 s no
less than the group's largest magnitude; a channel is stored as the whole number n in -7..7 next to x / s (ties to even) and
stands for n s.  Three operators work on such a cache:

  write      new tokens' rows (views of a projection's rows) are quantised into the slots of their pages; what the slots then
             stand for is read back, so that a pass returns its updated state
  read       the rows of listed slots as dense bf16 rows
  attention  every new token of a batch of sequences over its sequence's pages: single tokens, a few tokens at once (drafts
             to verify), prompts and later portions of prompts, batches of both; causal, with or without a window

Batches hold ``decodes`` sequences that get ``each`` tokens, and behind them ``prompts`` prompts (or next portions, where
``context`` tokens of each are stored already) with ``tokens`` tokens together.  Lengths are ragged and odd around the sizes
that a case names, pages lie scattered in the cache.
"""
from __future__ import annotations

import math
import random
import zlib

import torch

own = False

GROUP, MOST = 32, 7
HEADS = [(32, 8), (64, 8), (32, 4), (16, 4), (28, 4), (16, 16), (8, 1), (6, 2)]


def _store(name, op, tokens, heads, dim, page, pad=0):
    return {"name": name, "op": op, "tokens": tokens, "heads": heads[0], "kv_heads": heads[1], "dim": dim, "page": page, "pad": pad}


def _attend(name, heads, dim, page, decodes=0, decode_context=0, each=1, prompts=0, tokens=0, context=0, window=0):
    return {"name": name, "op": "attention", "heads": heads[0], "kv_heads": heads[1], "dim": dim, "page": page, "decodes": decodes,
            "decode_context": decode_context, "each": each, "prompts": prompts, "tokens": tokens, "context": context,
            "window": window}


def listed():
    return [
        _store("write 1", "write", 1, (32, 8), 128, 128),                # a single user's decode step: latency
        _store("write 777", "write", 777, (14, 2), 64, 16, pad=23),      # a small model's step, padded behind its tokens
        _store("write 8192", "write", 8192, (64, 8), 128, 128),          # a full step of prompts
        _store("read 1337", "read", 1337, (32, 8), 128, 128),            # one sequence's pages handed over
        _store("read 96000", "read", 96000, (32, 8), 128, 128),          # a batch's pages handed over
        _attend("decode 1", (32, 8), 128, 128, 1, 1337),                 # one user waiting for the next token: latency
        _attend("decode 256", (32, 8), 128, 128, 256, 1152),             # steady state of offline batches
        _attend("decode 3 long", (64, 8), 128, 128, 3, 60001),           # few users with long documents
        _attend("verify 40", (32, 4), 128, 128, 40, 2300, each=4),       # drafts of three tokens to verify
        _attend("prompt 137", (32, 8), 128, 128, prompts=1, tokens=137),      # a short question: time to first token
        _attend("mixed 8192", (32, 8), 128, 128, 192, 1100, prompts=8, tokens=8000),     # a full step of an offline batch
        _attend("portions 2000", (28, 4), 64, 16, prompts=3, tokens=2000, context=9000, window=4096),  # chunked prompts, window
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, dim, page = rng.choice(HEADS), rng.choice([128, 128, 64]), rng.choice([16, 32, 64, 128, 128])
    op = rng.choice(["write", "read", "decode", "decode", "prompt", "prompt"])
    if op in ("write", "read"):
        c = _store("", op, _log(rng, 1, (65536 if op == "write" else 768000) // max(8, heads[1])), heads, dim, page)
        if rng.random() < 0.4:
            c["pad"] = _log(rng, 1, 256)
    else:
        c = _attend("", heads, dim, page)
        if op == "decode" or rng.random() < 0.3:
            c["decodes"] = _log(rng, 1, 256)
            most = 2_300_000 if op == "decode" else 1_000_000                # pairs of a stored token and a head
            c["decode_context"] = _log(rng, 1, max(2, min(60000, most // (c["decodes"] * heads[1]))))
            c["each"] = rng.choice([1, 1, 1, 2, 4, 5]) if op == "decode" else 1
        if op == "prompt":
            c["tokens"] = _log(rng, 2, 8000)
            c["prompts"] = _log(rng, 1, max(1, min(12, c["tokens"] // 8)))
            if rng.random() < 0.4:
                c["context"] = _log(rng, 16, 9000)
            most = 128_000_000 // heads[0]                                   # pairs of a query and a key
            while c["tokens"] * (c["context"] + c["tokens"] / c["prompts"]) > most:
                c["context"], c["prompts"] = c["context"] // 2, c["prompts"] + 1
        if rng.random() < 0.25:
            c["window"] = _log(rng, 1, 5000)
    del c["name"]
    return c


# ---------------------------------------------------------------- what a batch holds
def _lengths(c):
    """(new tokens, stored tokens) of every sequence, decodes first."""
    rng = random.Random("%(decodes)d %(decode_context)d %(each)d %(prompts)d %(tokens)d %(context)d" % c)

    def around(x, n):
        return [max(1, round(x * rng.uniform(0.6, 1.4))) if n > 1 else x for _ in range(n)]
    new, old = [c["each"]] * c["decodes"], around(c["decode_context"], c["decodes"])
    if c["prompts"]:
        share = around(1000, c["prompts"])
        cuts = [c["tokens"] * sum(share[:i]) // sum(share) for i in range(c["prompts"] + 1)]
        new += [max(1, b - a) for a, b in zip(cuts, cuts[1:])]
        old += around(c["context"], c["prompts"]) if c["context"] else [0] * c["prompts"]
    return new, old


def _gen(*what):
    g = torch.Generator(device="cuda")
    g.manual_seed(zlib.crc32(repr(what).encode()))
    return g


def _rows(c, n, g):
    """Projection rows [q | k | v], some channels of the keys far above the others, as trained models have them."""
    hq, hkv, d = c["heads"], c["kv_heads"], c["dim"]
    x = torch.empty((n, hq + 2 * hkv, d), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    gain = torch.ones(d, device="cuda")
    gain[torch.randperm(d, generator=g, device="cuda")[:d // 16]] = 5.0
    x[:, hq:hq + hkv] *= gain.to(x.dtype)
    x[:, hq + hkv:] *= 0.3
    return x.view(n, -1)


def _split(c, rows):
    hq, hkv, d, n = c["heads"], c["kv_heads"], c["dim"], len(rows)
    return (rows[:, :hq * d].view(n, hq, d), rows[:, hq * d:(hq + hkv) * d].view(n, hkv, d),
            rows[:, (hq + hkv) * d:].view(n, hkv, d))


def _inputs(c, seed):
    g = _gen(seed, sorted((k, v) for k, v in c.items() if k != "name"))
    page, x = c["page"], {}
    if c["op"] == "attention":
        new, old = _lengths(c)
        lens = [a + b for a, b in zip(new, old)]
        pages = [-(-n // page) for n in lens]
        x["lens"], x["new"] = lens, new
        x["q"] = _split(c, _rows(c, sum(new), g))[0]
    else:
        pages = [-(-(c["tokens"] + c["pad"]) // page)]
    total = sum(pages)
    x["blocks"] = total + 3
    ids = torch.randperm(total + 3, generator=g, device="cuda")[:total].int()
    if c["op"] == "attention":
        table = torch.zeros((len(lens), max(pages)), dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(pages):
            table[i, :n] = ids[at:at + n]
            at += n
        x["table"] = table
        kept = (x["blocks"]) * page                                  # every slot holds a row, the unused ones of other sequences
        slots = torch.arange(kept, device="cuda")
    else:
        slots = (ids.long().unsqueeze(1) * page + torch.arange(page, device="cuda")).reshape(-1)[:c["tokens"] + c["pad"]]
        slots = slots.clone()
        if c["pad"]:
            slots[c["tokens"]:] = -1
    x["slots"] = slots
    _, x["k"], x["v"] = _split(dict(c, heads=0) if c["op"] == "attention" else c,
                               _rows(dict(c, heads=0) if c["op"] == "attention" else c, len(slots), g))
    return x


def prepare(case, seed):
    x, c = _inputs(case, seed), case
    state = {"case": c, "slots": x["slots"]}
    if own:
        from vllm_ascend_b200 import ops
        state["cache"] = tuple(ops.alloc_kv_cache_int4(x["blocks"], c["page"], c["kv_heads"], c["dim"], x["k"].device) for _ in "kv")
        if c["op"] != "write":
            ops.write_kv_int4(x["k"], x["v"], *state["cache"], x["slots"])
    else:
        n = x["blocks"] * c["page"]
        state["cache"] = tuple((torch.zeros((n, c["kv_heads"], c["dim"] // 2), dtype=torch.uint8, device="cuda"),
                                torch.zeros((n, c["kv_heads"], c["dim"] // GROUP), dtype=torch.bfloat16, device="cuda")) for _ in "kv")
        if c["op"] != "write":
            for cache, rows in zip(state["cache"], (x["k"], x["v"])):
                _put(cache, rows, x["slots"])
    if c["op"] == "write":
        state["k"], state["v"] = x["k"], x["v"]
    if c["op"] == "attention":
        state.update(q=x["q"], table=x["table"], new=x["new"], lens=x["lens"])
        if own:
            from vllm_ascend_b200.attention.metadata import metadata_from_tensors
            starts = torch.tensor([0] + x["new"], device="cuda").cumsum(0).int()
            state["meta"] = metadata_from_tensors(starts, torch.tensor(x["lens"], dtype=torch.int32, device="cuda"), x["table"],
                                                  max(x["new"]), max(x["lens"]), c["heads"], c["kv_heads"], c["dim"])
    return state


# ---------------------------------------------------------------- plain forms
def _quantise(x):
    """[..., channels] -> whole numbers and scales (fp32)."""
    g = x.float().unflatten(-1, (-1, GROUP))
    low = g.abs().amax(-1, keepdim=True)
    low = low / torch.full_like(low, MOST)
    s = ((low.view(torch.int32) + 0x7ffff) & ~0x7ffff).view(torch.float32)      # up to the next number of five bits
    n = torch.where(s > 0, g / torch.where(s > 0, s, 1.0), 0.0).round()
    return n, s


def _put(cache, rows, slots):
    codes, scales = cache
    n, s = _quantise(rows)
    n = (n.flatten(-2) + 8).to(torch.uint8)
    valid = slots >= 0
    at = slots[valid]
    codes[at] = (n[..., 0::2] | n[..., 1::2] << 4)[valid]
    scales[at] = s.squeeze(-1)[valid].to(torch.bfloat16)


def _get(cache, at):
    codes, scales = cache[0][at], cache[1][at]
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8
    return (n.unflatten(-1, (-1, GROUP)) * scales.float().unsqueeze(-1)).flatten(-2)


def _read(cache, slots):
    rows = _get(cache, slots.clamp_min(0))
    return torch.where((slots >= 0).view(-1, 1, 1), rows, 0.0).to(torch.bfloat16)


def _attention(state):
    c, q = state["case"], state["q"]
    group, page = c["heads"] // c["kv_heads"], c["page"]
    out, row = torch.empty(q.shape, dtype=q.dtype, device=q.device), 0
    for i, (new, n) in enumerate(zip(state["new"], state["lens"])):
        first = max(0, n - new - c["window"] + 1) if c["window"] else 0
        pos = torch.arange(first, n, device=q.device)
        at = state["table"][i][pos // page].long() * page + pos % page
        k, v = (_get(t, at).repeat_interleave(group, 1).transpose(0, 1) for t in state["cache"])         # [heads, keys, channels]
        for a in range(0, new, 1024):
            b = min(new, a + 1024)
            s = q[row + a:row + b].float().transpose(0, 1) @ k.transpose(1, 2) * c["dim"] ** -0.5
            mine = torch.arange(n - new + a, n - new + b, device=q.device).unsqueeze(1)
            hidden = pos > mine
            if c["window"]:
                hidden |= pos <= mine - c["window"]
            s.masked_fill_(hidden, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            out[row + a:row + b] = (p @ v / p.sum(-1, keepdim=True)).transpose(0, 1).to(q.dtype)
        row += new
    return out


def run(state):
    c = state["case"]
    if own:
        from vllm_ascend_b200 import ops
        k_cache, v_cache = state["cache"]
        if c["op"] == "attention":
            return ops.paged_attention_int4(state["q"], k_cache, v_cache, state["meta"], c["dim"] ** -0.5, window=c["window"])
        if c["op"] == "write":
            ops.write_kv_int4(state["k"], state["v"], k_cache, v_cache, state["slots"])
        return ops.read_kv_int4(k_cache, v_cache, state["slots"], c["dim"])
    if c["op"] == "attention":
        return _attention(state)
    if c["op"] == "write":
        for cache, rows in zip(state["cache"], (state["k"], state["v"])):
            _put(cache, rows, state["slots"])
    return tuple(_read(cache, state["slots"]) for cache in state["cache"])


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    stored = c["kv_heads"] * (c["dim"] // 2 + 2 * (c["dim"] // GROUP)) * 2            # bytes of a token's keys and values
    dense = c["kv_heads"] * c["dim"] * 2 * 2
    if c["op"] != "attention":
        rows, n = c["tokens"] + c["pad"], c["tokens"]
        if c["op"] == "write":
            return {"bytes": n * (dense + 2 * stored) + rows * (dense + 16), "flops": 4 * n * c["kv_heads"] * c["dim"] * 2}
        return {"bytes": n * stored + rows * (dense + 8), "flops": n * c["kv_heads"] * c["dim"] * 2}
    nbytes = pairs = 0
    for new, old in zip(*_lengths(c)):
        n, w = new + old, c["window"]
        nbytes += stored * (min(n, new + w - 1) if w else n) + 2 * new * c["heads"] * c["dim"] * 2
        pairs += sum(min(w, p) for p in range(old + 1, n + 1)) if w else new * old + new * (new + 1) // 2
    return {"bytes": nbytes, "flops": 4 * pairs * c["heads"] * c["dim"]}


# ---------------------------------------------------------------- in 64 bits, from the definition
def _stands_for(x):
    g = x.double().unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1, keepdim=True) / torch.tensor(7.0, dtype=torch.float64, device=x.device)
    _, e = torch.frexp(top)
    unit = torch.ldexp(torch.ones_like(top), e - 5)                   # of a number with five significant bits
    s = torch.ceil(top / unit) * unit
    s[top == 0] = 1.0
    return (torch.round(g / s) * s).flatten(-2)


def exact(case, seed):
    c, x = case, _inputs(case, seed)
    k, v = _stands_for(x["k"]), _stands_for(x["v"])
    if c["op"] != "attention":
        none = x["slots"] < 0
        k[none], v[none] = 0.0, 0.0
        return k, v
    q, outs, row = x["q"].double(), [], 0
    per = c["heads"] // c["kv_heads"]
    for i, (new, n) in enumerate(zip(x["new"], x["lens"])):
        keys = torch.arange(n, device=q.device)
        at = x["table"][i].long()[keys // c["page"]] * c["page"] + keys % c["page"]
        for a in range(0, new, 512):
            b = min(new, a + 512)
            own_pos = torch.arange(n - new + a, n - new + b, device=q.device)
            seen = keys[None] <= own_pos[:, None]
            if c["window"]:
                seen &= keys[None] > own_pos[:, None] - c["window"]
            rows = q[row + a:row + b].unflatten(1, (c["kv_heads"], per))
            s = torch.einsum("tghd,kgd->ghtk", rows, k[at]) / math.sqrt(c["dim"])
            p = torch.softmax(torch.where(seen, s, -math.inf), -1)
            outs.append(torch.einsum("ghtk,kgd->tghd", p, v[at]).flatten(1, 2))
        row += new
    return torch.cat(outs)
