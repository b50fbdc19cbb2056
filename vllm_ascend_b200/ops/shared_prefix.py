"""Attention of a batch whose sequences share prefixes: beams of one prompt, requests behind one system prompt, questions about one document.

The keys and values of a shared prefix are read once for all sequences of a group, each sequence's own keys behind it once for that
sequence, and both are joined.  The reference's platform turns its host's counterpart (cascade attention) off
(vllm_ascend/platform.py, ``_fix_incompatible_config``)."""
from __future__ import annotations

import struct
from ctypes import c_char_p
from dataclasses import dataclass
from typing import Optional

import torch

from .. import _native
from . import reference as ref
from .kv_int4 import _dense, _dense_heads, _elsewhere, _report

# laid out as the source's PlanArgs and SharedArgs
_PLAN = struct.Struct("@7P8i")
_ATTENTION = struct.Struct("@9P9qf9i")
for _name in ("b200_shared_plan", "b200_attn_shared"):
    _native.register_signature(_name, [c_char_p])

HEAD_SIZES = (64, 128)
#: ints of a base, query rows of one at most
_BASE, _ROWS = 12, 256


def has_kernel(dtype: torch.dtype, head_size: int, block_size: int) -> bool:
    """Whether queries and caches of that type, heads and pages of that size run the kernel on a GPU."""
    return dtype is torch.bfloat16 and head_size in HEAD_SIZES and block_size >= 8 and not (128 % block_size if block_size < 128 else block_size % 128)


@dataclass
class SharedPrefixPlan:
    """Which sequences share which prefix, and how the work is dealt out; made once a step for all layers of one head layout."""
    group_starts: torch.Tensor            # int32 [groups + 1] first sequence of each group
    prefix_lens: torch.Tensor             # int32 [groups]
    heads: int
    kv_heads: int
    tokens: int                           # query rows that belong to sequences, at most
    seqs: int
    blocks: int = 0
    bases_at: int = 0
    bases: int = 0
    table: Optional[torch.Tensor] = None
    stream: int = 0                                  # it was made on
    starts: Optional[torch.Tensor] = None            # the batch's own tensors: first query rows, lengths
    lens: Optional[torch.Tensor] = None

    def of(self, meta) -> bool:
        """Whether it was made for this batch, not for one that a copy of its metadata stands for."""
        return meta.query_start_loc is self.starts and meta.seq_lens is self.lens and meta.num_reqs == self.seqs


def plan_shared_prefix(meta, group_starts, prefix_lens, heads: int, kv_heads: int) -> SharedPrefixPlan:
    """Plan for ``paged_attention_shared`` over the batch of ``meta``: group g is sequences ``group_starts[g]`` up to ``group_starts[g + 1]``
    (int32 [groups + 1], in order; sequences in front of the first and behind the last group share nothing), and its first ``prefix_lens[g]`` keys
    are the same for all of them: they are read through the group's first sequence's row of the block table.  A prefix that reaches into new
    tokens counts up to where they begin.

    Lengths are read on the device: a captured plan follows what replays find there, as long as sequences, groups and query rows are no more than
    at capture.  Starts that are out of order or out of range, and lengths beyond what any cache holds, are reported through the status word, and nothing is
    computed.  A plan belongs to the stream that it is made on; calls on others wait for that one first."""
    device = meta.query_start_loc.get_device()
    if _elsewhere(device):
        with torch.cuda.device(device):
            return plan_shared_prefix(meta, group_starts, prefix_lens, heads, kv_heads)
    if kv_heads < 1 or heads < kv_heads or heads % kv_heads or heads // kv_heads > 128:
        raise ValueError(f"{heads} query heads do not share {kv_heads} heads of a cache evenly, 128 each at most")
    where = meta.query_start_loc.device
    starts, prefixes = (t if torch.is_tensor(t) else torch.tensor(t, dtype=torch.int32, device=where) for t in (group_starts, prefix_lens))
    if not (starts.dtype is prefixes.dtype is torch.int32 and starts.dim() == prefixes.dim() == 1 and starts.shape[0] == prefixes.shape[0] + 1
            and starts.get_device() == prefixes.get_device() == device):
        raise ValueError(f"group starts int32 [groups + 1] and prefix lengths int32 [groups] on {where}, not {starts.dtype} {tuple(starts.shape)} on "
                         f"{starts.device} and {prefixes.dtype} {tuple(prefixes.shape)} on {prefixes.device}")
    given, meta = meta, _dense(meta, device)
    starts, prefixes = starts.contiguous(), prefixes.contiguous()
    plan = SharedPrefixPlan(starts, prefixes, heads, kv_heads, max(int(meta.num_actual_tokens), int(meta.num_input_tokens)), meta.num_reqs,
                            starts=given.query_start_loc, lens=given.seq_lens)
    if device < 0:
        return plan
    G, groups, n = heads // kv_heads, prefixes.shape[0], meta.num_reqs
    plan.blocks = _native.sm_count(device)
    plan.bases = bases = groups + n + 2 * (plan.tokens // (2 * (128 // G)))
    plan.bases_at = -(-(4 + 2 * plan.blocks + 2 * plan.tokens + groups) // 4) * 4
    plan.table = torch.empty(plan.bases_at + bases * (_BASE + 2 * kv_heads), dtype=torch.int32, device=where)
    plan.stream = _native.stream_ptr()
    rc = _native.lib().b200_shared_plan(_PLAN.pack(
        meta.query_start_loc.data_ptr(), meta.seq_lens.data_ptr(), starts.data_ptr(), prefixes.data_ptr(), plan.table.data_ptr(),
        _native.status_word(where).data_ptr(), plan.stream, n, groups, plan.tokens, G, kv_heads, plan.blocks, bases, plan.bases_at))
    _native.check(rc, "shared_plan")
    _native.count_launch()
    return plan


def paged_attention_shared(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, meta, plan: SharedPrefixPlan, scale: float,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal ``paged_attention`` of q [T, Hq, D] over caches [blocks, tokens, heads, D] with the prefixes of ``plan`` read once a group.  Any number of
    new tokens a sequence.  Rows of ``out`` behind the last sequence are left as they are; a token without keys gets zeros.  bf16 with heads of
    64 and 128 runs the kernel, with 16 (D + 2) bytes of workspace for every row and query head; other types and sizes the definition.  Keys and values of pages that lie outside of a sequence may hold anything,
    those of its own new tokens are numbers."""
    shape, pages, device = q.shape, k_cache.shape, q.get_device()
    if len(shape) != 3 or len(pages) != 4 or v_cache.shape != pages or pages[3] != shape[2]:
        raise ValueError(f"queries [T, heads, D] and caches [blocks, tokens, heads, D], not {tuple(shape)}, {tuple(pages)} and {tuple(v_cache.shape)}")
    if _elsewhere(device):
        with torch.cuda.device(device):
            return paged_attention_shared(q, k_cache, v_cache, meta, plan, scale, out)
    (T, Hq, D), (NB, bs, Hkv, _) = shape, pages
    if Hq != plan.heads or Hkv != plan.kv_heads:
        raise ValueError(f"{Hq} heads on {Hkv}, a plan for {plan.heads} on {plan.kv_heads}")
    dtype = q.dtype
    if not dtype == k_cache.dtype == v_cache.dtype:
        raise ValueError(f"queries {dtype}, keys {k_cache.dtype} and values {v_cache.dtype} are not of one type")
    if not k_cache.get_device() == v_cache.get_device() == plan.prefix_lens.get_device() == device:
        raise ValueError(f"queries on {q.device}, caches on {k_cache.device} and {v_cache.device}, the plan on {plan.prefix_lens.device}")
    if not scale > 0:
        raise ValueError(f"scale {scale} is not above zero")
    n = meta.num_reqs
    if n != plan.seqs:
        raise ValueError(f"{n} sequences, a plan for {plan.seqs}")
    if T < plan.tokens and T < int(meta.query_start_loc_cpu[n]):
        raise ValueError(f"{T} query rows, a plan for {plan.tokens}")
    given = out
    if out is None:
        out = q.new_empty(shape)
    elif out.shape != shape or out.dtype != dtype or out.get_device() != device:
        raise ValueError(f"out: {dtype} {tuple(shape)} on {q.device}, not {out.dtype} {tuple(out.shape)} on {out.device}")
    if device < 0 or not has_kernel(dtype, D, bs):
        return _definition(q, k_cache, v_cache, _dense(meta, device), plan, scale, out)
    if T == 0 or plan.tokens == 0 or n == 0:
        return out
    table = meta.block_table
    if not (table.dtype is torch.int32 and table.dim() == 2 and table.stride(1) == 1 and table.shape[0] >= n and table.get_device() == device):
        table = _dense(meta, device).block_table
    q, k_cache, v_cache = _dense_heads(q), _as_pages(k_cache), _as_pages(v_cache)
    strides = k_cache.stride()
    if strides != v_cache.stride():
        v_cache = torch.empty_strided(pages, strides, dtype=dtype, device=v_cache.device).copy_(v_cache)
    if given is not None:
        row, head, channel = out.stride()
        if channel != 1 or head != D or row % 8 or out.data_ptr() % 16:
            out = q.new_empty(shape)
            out.copy_(given)
    stream = _native.stream_ptr()
    if stream != plan.stream:
        plan.table.record_stream(torch.cuda.current_stream())
    # every call has its own results of pieces: calls on two streams, or two graphs, may run at once
    part_rows = 4 * plan.tokens * Hq + plan.blocks * _ROWS
    parts = plan.prefix_lens.new_empty(part_rows * (D + 2))          # of 32 bits each
    rc = _native.lib().b200_attn_shared(_ATTENTION.pack(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), plan.table.data_ptr(), table.data_ptr(), parts.data_ptr(), out.data_ptr(),
        _native.status_word(plan.prefix_lens.device).data_ptr(), stream, q.stride(0), T, NB, table.stride(0), out.stride(0), part_rows,
        strides[0], strides[1], strides[2], scale, bs, table.shape[1], Hq, Hkv, D, plan.blocks, plan.tokens, plan.bases_at, plan.bases))
    _native.check(rc, "attn_shared")
    _native.count_launch(2)
    return out if given is None or out is given else given.copy_(out)


def _as_pages(cache: torch.Tensor) -> torch.Tensor:
    """The cache as tile copies read it: channels side by side, everything else on 16-byte boundaries."""
    block, token, head, channel = cache.stride()
    if channel == 1 and not (block % 8 or token % 8 or head % 8 or cache.data_ptr() % 16) and min(block, token, head) > 0:
        return cache
    return cache.contiguous()


def _definition(q, k_cache, v_cache, meta, plan, scale, out):
    table = meta.block_table[:meta.num_reqs]
    if q.is_cuda:
        NB, bs = k_cache.shape[:2]
        new = (meta.query_start_loc[1:meta.num_reqs + 1] - meta.query_start_loc[:meta.num_reqs]).unsqueeze(1)
        seen = (new > 0) & (torch.arange(table.shape[1], device=q.device) * bs < meta.seq_lens[:meta.num_reqs].unsqueeze(1))
        wrong = (table < 0) | (table >= NB)
        _report(wrong & seen, q.device)
        table = table.masked_fill(wrong, 0)
    return ref.paged_attention_shared(q, k_cache, v_cache, meta.query_start_loc_cpu, meta.seq_lens_cpu, table, plan.group_starts.tolist(),
                                      plan.prefix_lens.tolist(), scale, out)
