"""A paged cache of keys and values in 4 bits: allocation, the operators that fill and read it, attention over it.

Groups of 32 adjacent channels of a token and head share a scale of five significant bits; a channel is a whole number in
-7..7 times it, exact in bf16 (``reference.kv_int4_quantise``).  4.5 bits a channel: a GPU holds 3.5 times the tokens of a bf16
cache, and decode reads 3.5 times fewer bytes.  A cache is one dense uint8 tensor [blocks, heads, bytes of
a block] for the keys and one for the values, each at an address that 16 divides (layout: csrc/kv_int4.cuh); head sizes 64 and 128, blocks of a
multiple of 16 tokens.
The reference quantises its cache to 8 bits with static scales (vllm_ascend/quantization/methods/kv_c8.py)."""
from __future__ import annotations

import copy
import functools
import struct
from ctypes import c_char_p
from typing import Optional

import numpy as np
import torch

from .. import _native
from ..batch_invariant import fixed_sums
from . import reference as ref

# arguments go by address, laid out as the sources' Kv4Args and Int4Args: packing them takes 0.3 us where ctypes takes 0.1 us for each
_ROWS = struct.Struct("@7P4q3i")
_ATTENTION = struct.Struct("@10P6qf10i")
for _name in ("b200_kv_int4_write", "b200_kv_int4_read", "b200_attn_int4", "b200_attn_int4_prefill"):
    _native.register_signature(_name, [c_char_p])

HEAD_SIZES = (64, 128)
#: rows (new tokens times heads of a group) of a sequence up to which the kernel for few rows always takes it
FEW_ROWS = 32


def block_bytes(block_size: int, dim: int) -> int:
    """Bytes of a block of one head, of the keys or of the values."""
    if dim not in HEAD_SIZES:
        raise ValueError(f"a 4-bit cache takes heads of {HEAD_SIZES}, not {dim}")
    if block_size < 1 or block_size % ref.KV_INT4_TOKENS:
        raise ValueError(f"a 4-bit cache takes blocks of a multiple of {ref.KV_INT4_TOKENS} tokens, not {block_size}")
    return block_size // ref.KV_INT4_TOKENS * 9 * dim


def alloc_kv_cache_int4(num_blocks: int, block_size: int, heads: int, dim: int, device, arena=None) -> torch.Tensor:
    """Zero-filled cache [blocks, heads, bytes]; ``arena`` as in ``alloc_kv_cache``."""
    shape = (num_blocks, heads, block_bytes(block_size, dim))
    return arena.take(shape, torch.uint8) if arena is not None else torch.zeros(shape, dtype=torch.uint8, device=device)


def _check_caches(k_cache: torch.Tensor, v_cache: torch.Tensor, dim: int, device: int) -> tuple[int, int, int, int, int]:
    """Blocks, heads, block size and addresses of a pair of caches that belong together, on the device of that index (-1: the host), where bulk
    copies can read them."""
    shape, k_at, v_at = k_cache.shape, k_cache.data_ptr(), v_cache.data_ptr()
    if dim in HEAD_SIZES and len(shape) == 3 and shape[2] and shape[2] % (9 * dim) == 0 and v_cache.shape == shape \
            and k_cache.dtype is v_cache.dtype is torch.uint8 and k_cache.is_contiguous() and v_cache.is_contiguous() \
            and k_cache.get_device() == v_cache.get_device() == device and (k_at | v_at) & 15 == 0:
        return shape[0], shape[1], shape[2] // (9 * dim) * ref.KV_INT4_TOKENS, k_at, v_at
    if dim not in HEAD_SIZES:
        raise ValueError(f"a 4-bit cache takes heads of {HEAD_SIZES}, not {dim}")
    bs = ref.kv_int4_block_size(k_cache, dim)
    if v_cache.shape != shape or ref.kv_int4_block_size(v_cache, dim) != bs:
        raise ValueError(f"keys {tuple(shape)} and values {tuple(v_cache.shape)} are caches of different sizes")
    if not k_cache.get_device() == v_cache.get_device() == device:
        raise ValueError(f"caches on {k_cache.device} and {v_cache.device}, rows on device {device}")
    raise ValueError("a 4-bit cache begins on 16 bytes: bulk copies read it")


def _check_slots(slots: torch.Tensor, rows: int, device: int) -> torch.Tensor:
    if slots.dim() != 1 or slots.shape[0] != rows or slots.get_device() != device or slots.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"slots: {rows} whole numbers on device {device}, not {slots.dtype} {tuple(slots.shape)} on {slots.device}")
    return slots if slots.dtype is torch.int64 and slots.is_contiguous() else slots.to(torch.int64).contiguous()


def _dense_heads(x: torch.Tensor) -> torch.Tensor:
    """x [T, H, D] as the kernels read rows: heads dense, rows and the first element on 16-byte boundaries."""
    row, head, channel = x.stride()
    if channel == 1 and (head == x.shape[2] or x.shape[1] == 1) and row % 8 == 0 and x.data_ptr() % 16 == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _report(wrong: torch.Tensor, device: torch.device) -> None:
    """Sets the device's status word where an index is out of range, as the kernels do.  An indexing operator would end the process's
    work on that GPU."""
    _native.status_word(device).masked_fill_(wrong.any(), _native.BAD_INDEX)


def _elsewhere(device: int) -> bool:
    """Whether tensors of that device index are on a GPU that is not the current one."""
    return device >= 0 and device != torch.cuda.current_device()


def write_kv_int4(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Rows of k and v [T, heads, D] quantised into their slots (block * block size + offset) of a 4-bit cache; rows whose slot
    is below zero are not stored.  A slot may be listed once only."""
    if k.dim() != 3 or k.shape != v.shape or k.dtype != v.dtype or not k.is_floating_point() or k.get_device() != v.get_device():
        raise ValueError(f"keys {k.dtype} {tuple(k.shape)} and values {v.dtype} {tuple(v.shape)} are not rows [T, heads, D] of one type")
    T, H, D = k.shape
    device = k.get_device()
    if _elsewhere(device):
        with torch.cuda.device(device):
            return write_kv_int4(k, v, k_cache, v_cache, slot_mapping)
    NB, heads, bs, k_at, v_at = _check_caches(k_cache, v_cache, D, device)
    if H != heads:
        raise ValueError(f"rows of {H} heads, a cache of {heads}")
    slots = _check_slots(slot_mapping, T, device)
    if T == 0:
        return
    if device < 0 or k.dtype is not torch.bfloat16:
        if device >= 0:
            beyond = slots >= NB * bs
            _report(beyond, k.device)
            slots = slots.masked_fill(beyond, -1)
        return ref.write_kv_int4(k, v, k_cache, v_cache, slots)
    k, v = _dense_heads(k), _dense_heads(v)
    rc = _native.lib().b200_kv_int4_write(_ROWS.pack(
        k.data_ptr(), v.data_ptr(), slots.data_ptr(), k_at, v_at, _native.status_word(k.device).data_ptr(),
        _native.stream_ptr(), k.stride(0), v.stride(0), T, NB * bs, H, D, bs))
    _native.check(rc, "kv_int4_write")
    _native.count_launch()


def read_kv_int4(k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, dim: int) -> tuple[torch.Tensor, torch.Tensor]:
    """What slots of a 4-bit cache of heads of ``dim`` stand for: keys and values [slots, heads, dim] in bf16, exact.  Slots below zero
    read as zeros; a slot may be listed any number of times."""
    device = k_cache.get_device()
    if _elsewhere(device):
        with torch.cuda.device(device):
            return read_kv_int4(k_cache, v_cache, slots, dim)
    NB, H, bs, k_at, v_at = _check_caches(k_cache, v_cache, dim, device)
    n = slots.shape[0] if slots.dim() else 0
    slots = _check_slots(slots, n, device)
    if device < 0:
        return ref.read_kv_int4(k_cache, v_cache, slots, dim)
    k = k_cache.new_empty((n, H, dim), dtype=torch.bfloat16)
    v = torch.empty_like(k)
    if n == 0:
        return k, v
    rc = _native.lib().b200_kv_int4_read(_ROWS.pack(
        k.data_ptr(), v.data_ptr(), slots.data_ptr(), k_at, v_at, _native.status_word(k.device).data_ptr(),
        _native.stream_ptr(), H * dim, H * dim, n, NB * bs, H, dim, bs))
    _native.check(rc, "kv_int4_read")
    _native.count_launch()
    return k, v


#: parts whose blocks form a cluster and join in it
CLUSTER = 16
#: us that a pair of query tiles takes to start and end, and a tile of 128 keys of one query tile (two: a quarter more), by head size
PAIR_US = 7.5
TILE_US = {128: 1.9, 64: 1.5}


def _parts(blocks: int, max_len: int, at_once: int, known: bool) -> int:
    """Parts that every sequence's keys are split into, by the blocks without a split and those that run at once.  Clusters of more than eight
    find room where there are few, and pay for long sequences; more parts than a cluster's join in a second kernel, 6 us more.  32 heads on 8,
    one sequence of 1337 tokens 6.2 us in 8 parts, 7.2 in 16, 12 in 18; of 12000 13.4, 11.8, 15.9; of 40000 31, 25, 24; four of 8000 15 in 8,
    19.5 in 12.  64 on 8, three of 60000 76 in 8, 61 in 14, 58 in 18, the most that was tried; all with heads of 128.  In a graph (lengths not
    ``known``) ``max_len`` is what the table holds; a quarter of it counts."""
    if fixed_sums():
        return 1
    most, wide = min(at_once // max(1, blocks), -(-max_len // 128), 18), 16 if blocks <= 8 else 14
    if most > CLUSTER and known and max_len > 40000:
        return most
    if most >= wide and blocks * 18 <= at_once and (max_len if known else max_len / 4) >= 8000:
        return wide
    return max(1, min(most, 8))


def _parts_of_rounds(blocks: int, max_len: int, mean: float, at_once: int, D: int) -> int:
    """The same for lengths that the host knows, where the blocks without a split fill more than half of the GPU: those that take least time,
    a block in 5 us and its tokens' time, half a round for the last ones of unequal lengths, 3 us for a cluster's joins.  32 heads on 8 of 128: 30
    sequences of about 8000 85 us whole, 71 in three; 64 of them 141 and 124 in two; 96 of 2000 55, 61 in two."""
    token = 0.01 if D == 128 else 0.0065

    def us(parts):
        rounds = blocks * parts / at_once
        if rounds <= 1:
            return 5 + max(0.72, 0.5 + 0.5 * rounds) * token * max_len / parts + 3 * (parts > 1)
        return (rounds + 0.5) * (5 + token * mean / parts) + 3 * (parts > 1)
    return min(range(1, 9), key=us)


def paged_attention_int4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, meta, scale: float,
                         out: Optional[torch.Tensor] = None, causal: bool = True, window: int = 0) -> torch.Tensor:
    """``paged_attention`` over a 4-bit cache: q [T, Hq, D], every new token over its sequence's pages.  Rows of ``out`` behind the last
    sequence are left as they are; a token that sees no key gets zeros."""
    if q.dim() != 3:
        raise ValueError(f"queries are [T, heads, D], not {tuple(q.shape)}")
    T, Hq, D = q.shape
    device = q.get_device()
    if _elsewhere(device):
        with torch.cuda.device(device):
            return paged_attention_int4(q, k_cache, v_cache, meta, scale, out, causal, window)
    NB, Hkv, bs, k_at, v_at = _check_caches(k_cache, v_cache, D, device)
    if Hkv == 0 or Hq % Hkv or Hq == 0:
        raise ValueError(f"{Hq} query heads do not share {Hkv} heads of a cache evenly")
    if not scale > 0:
        raise ValueError(f"scale {scale} is not above zero")
    if window < 0:
        raise ValueError(f"window {window} is below zero")
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((T, Hq, D))
    elif out.shape != q.shape or out.dtype != q.dtype or out.get_device() != device:
        raise ValueError(f"out: {q.dtype} {tuple(q.shape)} on {q.device}, not {out.dtype} {tuple(out.shape)} on {out.device}")
    n = meta.num_reqs
    cu, lens, table = meta.query_start_loc, meta.seq_lens, meta.block_table
    pages, strides = table.shape, table.stride()
    if not (cu.dtype is lens.dtype is table.dtype is torch.int32 and cu.get_device() == lens.get_device() == table.get_device() == device
            and cu.stride() == lens.stride() == (1,) and len(strides) == 2 and strides[1] == 1 and cu.numel() > n and lens.numel() >= n
            and pages[0] >= n):
        meta = _dense(meta, device)
        cu, lens, table = meta.query_start_loc, meta.seq_lens, meta.block_table
        pages, strides = table.shape, table.stride()
    if device < 0 or q.dtype is not torch.bfloat16:
        if device >= 0:
            table = _pages_in_range(cu, lens, table[:n], NB, bs, window)
        return ref.paged_attention_int4(q, k_cache, v_cache, meta.query_start_loc_cpu, meta.seq_lens_cpu, table, scale, causal, window, out=out)
    if n == 0 or T == 0:
        return out
    given, q = out, _dense_heads(q)
    row, head, channel = out.stride()
    if channel != 1 or head != D or row % 8 or out.data_ptr() % 16:
        out = q.new_empty((T, Hq, D))
        out.copy_(given)
    max_q, G = meta.max_query_len, Hq // Hkv
    window = min(window, 2 ** 31 - 1 - T)            # the first key of a window in 32 bits: positions are -T at least
    args = (q, k_at, v_at, NB, Hkv, meta, pages[1], strides[0], scale, out, causal, window, bs)
    if max_q * G <= FEW_ROWS or G > 128:
        _few_rows(*args, 0, n, max_q)
    else:
        starts, keys = meta.query_start_loc_cpu, meta.seq_lens_cpu
        for few, first, end, what in _plan(starts.tobytes(), starts.dtype.char, keys.tobytes(), keys.dtype.char, n, window, G, Hkv, D,
                                           _native.sm_count(device), fixed_sums()):
            if few:
                _few_rows(*args, first, end, what[0])
            else:
                _prompts(*args, first, end, *what)
    return out if out is given else given.copy_(out)


def _dense(meta, device: int):
    """Metadata as the kernels walk it: row numbers and lengths without gaps, tables whose rows have none."""
    n, cu, lens, table = meta.num_reqs, meta.query_start_loc, meta.seq_lens, meta.block_table
    if not (cu.dtype is lens.dtype is table.dtype is torch.int32 and cu.get_device() == lens.get_device() == table.get_device() == device
            and cu.dim() == lens.dim() == 1 and table.dim() == 2 and cu.shape[0] > n and lens.shape[0] >= n and table.shape[0] >= n):
        raise ValueError(f"metadata of {n} sequences: row numbers {cu.dtype} {tuple(cu.shape)}, lengths {lens.dtype} {tuple(lens.shape)}, "
                         f"pages {table.dtype} {tuple(table.shape)}, not int32 on device {device}")
    meta = copy.copy(meta)
    meta.query_start_loc, meta.seq_lens, meta.block_table = cu.contiguous(), lens.contiguous(), table.contiguous()
    return meta


def _pages_in_range(cu, lens, table, blocks: int, bs: int, window: int) -> torch.Tensor:
    """The table with page 0 in place of what is no page; reported where a new token sees such a page."""
    n, columns = table.shape
    new, lens = (cu[1:n + 1] - cu[:n]).unsqueeze(1), lens[:n].unsqueeze(1)
    col = torch.arange(columns, device=table.device)
    seen = (new > 0) & (col * bs < lens)
    if window:
        seen &= (col + 1) * bs > lens.long() - new - window + 1
    wrong = (table < 0) | (table >= blocks)
    _report(wrong & seen, table.device)
    return table.masked_fill(wrong, 0)


def _few_us(new, keys, G: int, Hkv: int, D: int, sms: int) -> float:
    """About what a launch of the kernel for few rows takes in us for sequences with so many new tokens and keys: a block of 16 rows (two an
    SM at once) costs its start and its units of 16 keys, and every sequence has as many blocks as the longest.  Fitted like ``_prompt_us`` to
    prompts, portions and drafts of 8 to 1000 tokens."""
    blocks = -(-new * G // 16)
    units = float((blocks * ((keys - new / 2).clip(0) / 16 + 1)).sum()) * Hkv * (1 if D == 128 else 0.65)
    idle = (len(new) * int(blocks.max()) - int(blocks.sum())) * Hkv
    return 4 + (1.75 * int(blocks.sum()) * Hkv + 0.4 * idle + 0.1 * units) / sms


def _prompt_us(new, keys, G: int, Hkv: int, D: int, sms: int) -> float:
    """The same for the kernel for prompts: a pair of query tiles, one an SM, costs its start and its tiles of 128 keys.  32 heads on 8 of 128: 137
    tokens 7.7 us there, 11.6 here; 300 tokens 16.5 and 14.9; 30 behind 4000 17 and 24; 8 x 100 30 and 14; 40 x 8 behind 2000 80 and 112.
    64 on 8: 137 tokens 12.3 and 11.8, 40 x 8 behind 2000 126 and 112."""
    pairs = -(-new // (2 * (128 // G)))
    blocks = int(pairs.sum()) * Hkv
    parts = _prompt_parts(blocks, int(keys.max()), int(new.sum()), G * Hkv, D, sms)
    us = PAIR_US + TILE_US[D] / parts * ((keys - new / 2).clip(0) / 128 + 0.5) * np.where(new * G > 128, 1.25, 1)
    rounds = blocks * parts / sms
    return 1 + 5 * (parts > 1) + (float(us.max()) if rounds <= 1 else (rounds + 0.5) * float((us * pairs).sum()) * Hkv / blocks)


@functools.lru_cache(maxsize=256)
def _plan(cu: bytes, cu_type: str, lens: bytes, lens_type: str, n: int, window: int, G: int, Hkv: int, D: int, sms: int, fixed: bool) -> tuple:
    """Launches for ``n`` sequences that begin at these row numbers and have so many keys: (whether of the kernel for few rows, first sequence, end,
    and the most new tokens of one, or their rows and pairs of query tiles).  Sequences of few rows in front of the others go to the kernel for
    them; those behind go with the others, to the kernel that takes less time for them, or all go to that for few rows in one launch.  With
    sums in a fixed order (``fixed``) a sequence's kernel follows from its own rows alone."""
    new = np.diff(np.frombuffer(cu, dtype=cu_type)[:n + 1].astype(np.int64))
    many = new * G > FEW_ROWS
    if fixed:
        ends = (np.flatnonzero(np.diff(many)) + 1).tolist()
        runs = [(not many[a], a, b) for a, b in zip([0, *ends], [*ends, len(new)])]
    else:
        first = int(many.argmax()) if many.any() else n
        runs = [(True, 0, first)] if first else []
        if int(new[first:].sum()) * G * Hkv > 256 * sms:              # 16 blocks of 16 rows an SM: never near
            runs.append((False, first, n))
        elif first < n:
            shape, keys = (G, Hkv, D, sms), np.maximum(np.frombuffer(lens, dtype=lens_type)[:n].astype(np.int64), 0)
            if window:
                keys = np.minimum(keys, window + new)
            few, rest = _few_us(new[first:], keys[first:], *shape), _prompt_us(new[first:], keys[first:], *shape)
            runs.append((few < rest, first, n))
            if first and _few_us(new, keys, *shape) < min(few, rest) + _few_us(new[:first], keys[:first], *shape):
                runs = [(True, 0, n)]
    plan = []
    for few, a, b in runs:
        x = new[a:b]
        plan.append((few, a, b, (int(x.max()),) if few else (int(x.sum()), int((-(-x // (2 * (128 // G)))).sum()))))
    return tuple(plan)


def _few_rows(q, k_at, v_at, NB, Hkv, meta, columns, pitch, scale, out, causal, window, bs, first, end, max_q) -> None:
    """Sequences ``first`` to ``end``, none with more than ``max_q`` new tokens."""
    T, Hq, D = q.shape
    n = end - first
    rows = max_q * (Hq // Hkv)
    blocks = n * Hkv * (1 if rows <= 8 else -(-rows // 16))
    # a captured graph is replayed with other lengths, up to what the table holds
    capturing = torch.cuda.is_current_stream_capturing()
    longest, at_once = columns * bs if capturing else meta.max_seq_len, (3 if rows <= 8 else 2) * _native.sm_count(q.get_device())
    if window:
        longest = min(longest, window + max_q)
    if 2 * blocks <= at_once or longest < 2048 or capturing or fixed_sums():
        parts = _parts(blocks, longest, at_once, not capturing)
    else:
        parts = _parts_of_rounds(blocks, longest, min(float(meta.seq_lens_cpu[first:end].mean()), longest), at_once, D)
    ahead = T if end == meta.num_reqs else int(meta.query_start_loc_cpu[end])       # rows of these sequences and those in front of them
    if parts > CLUSTER and parts > _most_parts(ahead, Hq, D):
        parts = 8
    scratch = _results(q, ahead, parts) if parts > CLUSTER else None
    cu, lens, table = _of(meta, first)
    rc = _native.lib().b200_attn_int4(_ATTENTION.pack(
        q.data_ptr(), k_at, v_at, cu.data_ptr(), lens.data_ptr(), table.data_ptr(), out.data_ptr(),
        0 if scratch is None else scratch.data_ptr(), _native.status_word(q.device).data_ptr(), _native.stream_ptr(), q.stride(0), ahead, NB,
        out.stride(0), 0, pitch, scale, bs, columns, n, max_q, Hq, Hkv, D, int(causal), window, parts))
    _native.check(rc, "attn_int4")
    _native.count_launch(1 + int(parts > CLUSTER))


def _of(meta, first: int):
    """Row numbers, lengths and pages of the sequences from ``first`` on."""
    cu, lens, table = meta.query_start_loc, meta.seq_lens, meta.block_table
    return (cu[first:], lens[first:], table[first:]) if first else (cu, lens, table)


#: bytes of the parts' results of a call at most
MOST_BYTES = 256 << 20


def _most_parts(rows: int, heads: int, D: int) -> int:
    return MOST_BYTES // (max(rows, 1) * heads * (D + 1) * 4)


def _results(q, rows: int, parts: int) -> torch.Tensor:
    """Memory for the results of parts.  Each call has its own: calls on two streams, or two graphs, may run at once."""
    _, Hq, D = q.shape
    return torch.empty(rows * Hq * parts * (D + 1), dtype=torch.float32, device=q.device)


@functools.lru_cache(maxsize=1024)
def _prompt_parts(blocks: int, max_len: int, tokens: int, heads: int, D: int, sms: int) -> int:
    """Parts of a prompt's keys, of 512 at least: those that take least time in rounds of one block an SM, each of ``PAIR_US`` and its tiles, with
    a join that writes and reads the parts' fp32 results.  32 heads on 8 of 128, 1300 tokens behind 8000 (168 blocks): 278 us whole, 252 in three;
    600 behind 20000 (80 blocks): 339, 253; 64 on 8, 700 behind 20000 (176 blocks): 652, 498 in four; 28 on 4 of 64, 2000 behind 9000 in a window of
    4096 (232 blocks): 142, 168."""
    tiles, tile = max_len / 128, 1.25 * TILE_US[D]

    def us(parts):
        join = 5 + tokens * heads * D * 8 * parts / 4e6
        whole = -(-blocks * parts // sms) * (PAIR_US + tile * tiles / parts)
        return 1.08 * whole + join if parts > 1 else whole           # sequences of unequal lengths gain less
    return min(range(1, max(1, min(max_len // 512, 16)) + 1), key=us)


def _prompts(q, k_at, v_at, NB, Hkv, meta, columns, pitch, scale, out, causal, window, bs, first, end, tokens, pairs) -> None:
    """Sequences ``first`` to ``end`` with so many new tokens and pairs of query tiles."""
    T, Hq, D = q.shape
    longest = min(meta.max_seq_len, window + meta.max_query_len) if window else meta.max_seq_len
    parts = 1 if fixed_sums() else _prompt_parts(pairs * Hkv, longest, tokens, Hq, D, _native.sm_count(q.get_device()))
    if parts > 1 and parts > _most_parts(T, Hq, D):
        parts = 1
    scratch = _results(q, T, parts) if parts > 1 else None
    cu, lens, table = _of(meta, first)
    rc = _native.lib().b200_attn_int4_prefill(_ATTENTION.pack(
        q.data_ptr(), k_at, v_at, cu.data_ptr(), lens.data_ptr(), table.data_ptr(), out.data_ptr(),
        0 if scratch is None else scratch.data_ptr(), _native.status_word(q.device).data_ptr(), _native.stream_ptr(), q.stride(0), T, NB,
        out.stride(0), tokens, pitch, scale, bs, columns, end - first, 0, Hq, Hkv, D, int(causal), window, parts))
    _native.check(rc, "attn_int4_prefill")
    _native.count_launch(1 + int(parts > 1))
