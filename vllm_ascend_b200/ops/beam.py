"""Steps of a beam search on the device: the best continuations over all beams and the whole vocabulary, and the beams' states (recurrent
states, the pages that beams have of their own) brought behind the parents that were chosen.

``beam_select`` gives parents as ``reorder_beams`` takes them, so a step needs no copy to the host between the two.  The reference's host framework
sorts candidates on the host and starts every round with new requests (``LLM.beam_search`` on a batch of prompts)."""
from __future__ import annotations

import functools
import math
import struct
from ctypes import c_char_p
from typing import Optional, Sequence

import torch

from .. import _native
from . import reference as ref

# laid out as the source's SelectArgs, BeamTensor and ReorderArgs
_SELECT = struct.Struct("@11Pq8i")
_TENSOR = struct.Struct("@P4q4i")
_REORDER = struct.Struct("@6P5i")
for _name in ("b200_beam_select", "b200_beam_reorder"):
    _native.register_signature(_name, [c_char_p])

#: continuations of a group, beams of a group at most
MOST_SELECTED = 256
MOST_BEAMS = 1024
#: elements of a row that a block takes at a time
TILE = 4096
#: tokens of a vocabulary at most: positions of 32 bits count up to eight tiles past its end
MOST_TOKENS = 2 ** 31 - 1 - 8 * TILE


@functools.lru_cache(maxsize=4096)
def _parts(rows: int, vocab: int, sms: int) -> tuple[int, int]:
    """(parts, elements of a part) of every row: whole tiles, as many as run at once, two blocks an SM.  A block takes about 8 us to begin and to end
    and 0.5 us a tile: 64 rows of 151936 in 1, 2, 4, 8, 19 parts 34, 25, 24, 28, 46 us; 768 rows 107, 124, 134, 189, 381."""
    tiles = -(-(vocab + 7) // TILE)
    per = -(-tiles // max(1, min(tiles, 2 * sms // rows)))
    return -(-tiles // per), per * TILE


def beam_select(logits: torch.Tensor, scores: torch.Tensor, k: Optional[int] = None,
                dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``k`` best continuations of every group (default: two for each beam, so that as many as there are beams do not end).

    logits [groups * beams, vocabulary], rows in the order of ``scores``; scores [groups, beams], the log-probability of each beam so far,
    -inf for beams that ended (their logits are not read).  A continuation's total is its beam's score plus the token's log-probability.
    ``dtype``, fp32 or fp64, is the type of scores and totals: totals that become the next step's scores keep what was added up in 64 bits.
    Returns totals, parents (int32, a beam of the group) and tokens (int64), each [groups, k], best first; equal totals come in the order
    of beams, then tokens.  A row that holds a NaN or +inf, or nothing above -inf, has no distribution: its tokens count as -inf, like masked
    ones.  Exponentials and the sums that a thread adds up (a 512th of a row at most) are held in 32 bits, what they add up to and totals in 64: a total
    of a row of 151936 is off by 3e-8 as a rule and by less than 4e-6, continuations further apart than that come in the order of their exact totals."""
    if logits.dim() != 2 or scores.dim() != 2 or not logits.is_floating_point():
        raise ValueError(f"logits [groups * beams, vocabulary] and scores [groups, beams], not {logits.dtype} {tuple(logits.shape)} and "
                         f"{tuple(scores.shape)}")
    (rows, vocab), (groups, width), device = logits.shape, scores.shape, logits.get_device()
    if dtype not in (torch.float32, torch.float64):
        raise ValueError(f"scores and totals of {dtype}: fp32 or fp64")
    if rows != groups * width or scores.dtype != dtype or scores.get_device() != device:
        raise ValueError(f"{rows} rows of logits on {logits.device}, scores {scores.dtype} {tuple(scores.shape)} on {scores.device} for totals of {dtype}")
    if width < 1 or width > MOST_BEAMS or not 1 <= vocab <= MOST_TOKENS or width * vocab > 2 ** 31 - 1:
        raise ValueError(f"{width} beams over {vocab} tokens: 1 to {MOST_BEAMS} beams of up to {MOST_TOKENS} tokens, fewer than 2^31 candidates")
    if k is None:
        k = min(2 * width, width * vocab)
    if not 1 <= k <= min(MOST_SELECTED, width * vocab):
        raise ValueError(f"{k} of {width * vocab} continuations: 1 to {MOST_SELECTED}")
    if device < 0:
        return ref.beam_select(logits, scores, k)
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return beam_select(logits, scores, k, dtype)
    if logits.dtype not in (torch.bfloat16, torch.float32):
        logits = logits.float()                                 # 64-bit logits round to 32
    if logits.stride(1) != 1 and vocab > 1:
        logits = logits.contiguous()
    scores = scores.contiguous()
    totals = torch.empty((groups, k), dtype=dtype, device=logits.device)
    parents = torch.empty((groups, k), dtype=torch.int32, device=logits.device)
    tokens = torch.empty((groups, k), dtype=torch.int64, device=logits.device)
    if groups == 0:
        return totals, parents, tokens
    parts, per = _parts(rows, vocab, _native.sm_count(device))
    # every call has its own: calls on two streams, or two graphs, may run at once
    slots = rows * parts
    memory = torch.empty(slots * (k * 8 + 16), dtype=torch.uint8, device=logits.device)
    keys = memory.data_ptr()
    sums = keys + slots * k * 8
    maxima = sums + slots * 8
    rc = _native.lib().b200_beam_select(_SELECT.pack(
        logits.data_ptr(), scores.data_ptr(), keys, maxima + slots * 4, maxima, sums, totals.data_ptr(), parents.data_ptr(), tokens.data_ptr(),
        _native.status_word(logits.device).data_ptr(), _native.stream_ptr(), logits.stride(0), groups, width, vocab, k, parts, per,
        int(logits.dtype == torch.float32), int(dtype == torch.float64)))
    _native.check(rc, "beam_select")
    _native.count_launch(2)
    return totals, parents, tokens


class BeamStates:
    """Tensors that follow the beams, and where their rows lie; made by ``beam_states``."""

    def __init__(self, tensors: list, paged: bool, int4_dim: int):
        self.tensors, self.paged, self.int4_dim = tensors, paged, int4_dim
        self.device = tensors[0].device
        self._table, self._wide, self._stream = None, 0, 0
        rows = [_layout(t, paged, int4_dim) for t in tensors]
        _check_apart(rows)
        rows.sort(key=lambda r: -r[-1])
        if self.device.type == "cuda":
            packed = b"".join(_TENSOR.pack(*r) for r in rows)
            self._table = torch.frombuffer(bytearray(packed), dtype=torch.uint8).to(self.device)
            self._wide = sum(r[-1] == 16 for r in rows)
            with torch.cuda.device(self.device):
                self._stream = _native.stream_ptr()


def _layout(t: torch.Tensor, paged: bool, int4_dim: int) -> tuple:
    """How a row (or page) of a tensor lies in memory, as the kernel walks it."""
    size, quantised = t.element_size(), paged and t.dtype == torch.uint8
    if t.dim() != (3 if quantised else 4) if paged else t.dim() < 1:
        raise ValueError(f"rows, or pages [pages, tokens, heads, channels], not {tuple(t.shape)}")
    outer, run, tokens = 1, 0, 1
    if not paged:
        if t.shape[0] and not t[0].is_contiguous():
            raise ValueError(f"rows are dense: shape {tuple(t.shape)}, strides {t.stride()}")
        unit, units, tokens = (t[0].numel() if t.shape[0] else 0) * size, 1, 0
    elif quantised:                                             # [pages, heads, bytes], units of 16 tokens
        if int4_dim < 1 or t.shape[2] % (9 * int4_dim) or not t.is_contiguous():
            raise ValueError(f"a 4-bit cache of heads of {int4_dim}, dense: shape {tuple(t.shape)}, strides {t.stride()}")
        outer, run, tokens = t.shape[1], t.stride(1), ref.KV_INT4_TOKENS
        unit, units = 9 * int4_dim, t.shape[2] // (9 * int4_dim)
    else:
        _, units, heads, dim = t.shape
        if t.stride(3) != 1 and dim > 1:
            raise ValueError(f"channels lie side by side: strides {t.stride()}")
        if (t.stride(2) == dim or heads == 1) and (t.stride(1) == heads * dim or units == 1):      # a token's heads in one run
            unit = heads * dim * size
        elif (t.stride(1) == dim or units == 1) and t.stride(2) >= units * dim:                    # a head's tokens in one run
            outer, run, unit = heads, t.stride(2) * size, dim * size
        else:
            raise ValueError(f"pages hold a token's heads or a head's tokens in one run: shape {tuple(t.shape)}, strides {t.stride()}")
    row = t.stride(0) * size
    if t.shape[0] > 1 and row < (outer - 1) * run + units * unit:
        raise ValueError(f"rows overlap: shape {tuple(t.shape)}, strides {t.stride()}")
    width = 16
    while width > 1 and any(n % width for n in (t.data_ptr(), row, run, unit)):
        width //= 2
    return t.data_ptr(), row, run, unit, t.shape[0], outer, units, tokens, width


def _check_apart(rows: list) -> None:
    """Refuses memory that two tensors would move.  Rows may lie between each other's, as in slices of one buffer."""
    ordered = sorted(r for r in rows if r[4] and r[6] * r[3])
    for i, a in enumerate(ordered):
        end = a[0] + (a[4] - 1) * a[1] + (a[5] - 1) * a[2] + a[6] * a[3]
        for b in ordered[i + 1:]:
            if b[0] >= end:
                break
            if _meet(a, b):
                raise ValueError("two of the tensors share memory")


def _meet(a: tuple, b: tuple) -> bool:
    """Whether two layouts share memory, b not in front of a: exactly where rows and pieces are as far apart in both, else also where the places of
    rows, modulo what both distances between rows are multiples of, do not tell."""
    at, row, run, unit, n, outer, units, _, _ = a
    at2, row2, run2, unit2, n2, outer2, units2, _, _ = b
    one, two, off = units * unit, units2 * unit2, at2 - at               # bytes of a piece
    span, span2 = (outer - 1) * run + one, (outer2 - 1) * run2 + two
    if (row == row2 or n == 1 or n2 == 1) and (run == run2 or outer == 1 or outer2 == 1):
        row, run = (row2 if n == 1 else row) if n * n2 > 1 else 1, (run2 if outer == 1 else run) if outer * outer2 > 1 else 1
        # rows d apart whose extents meet, then their first pieces that end behind the other's begin
        for d in range(max(1 - n, (-span2 - off) // row), min(n2 - 1, (span - off) // row) + 1):
            apart = off + d * row
            j = max(1 - outer, (-two - apart) // run + 1)
            if j < outer2 and apart + j * run < one:
                return True
        return False
    every = math.gcd(row if n > 1 else 0, row2 if n2 > 1 else 0) or span + span2 + off
    off %= every
    return off < span or off + span2 > every


def beam_states(tensors: Sequence[torch.Tensor], paged: bool = False, int4_dim: int = 0) -> BeamStates:
    """Handle for ``reorder_beams``: tensors of any types and sizes on one device whose first dimension is a row (recurrent states) or, with
    ``paged``, a page (caches [pages, tokens, heads, channels] in either physical order, or 4-bit ones of heads of ``int4_dim``).  No two of them share
    memory.  It holds addresses: keep it as long as the tensors, make another when they are replaced."""
    tensors = list(tensors)
    if not tensors:
        raise ValueError("no tensors")
    if any(t.device != tensors[0].device for t in tensors):
        raise ValueError(f"tensors on {sorted({str(t.device) for t in tensors})}: one handle a device")
    return BeamStates(tensors, paged, int4_dim)


def reorder_beams(states: BeamStates, rows: torch.Tensor, parents: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> None:
    """In place, for all tensors of ``states`` in one launch: row ``rows[g, w]`` becomes what row ``rows[g, parents[g, w]]`` was before the call.

    rows, parents int32 [groups, beams]; a parent is a beam of the same group, -1 leaves the row as it is; row -1: the group has no such beam.  All
    rows of a call are different.  With pages, ``lengths`` (int32 [groups]) says how many tokens of a group's pages are filled: the rest of a page
    is left as it is.  Rows and parents out of range are reported through the status word and move nothing."""
    device = states.device.index if states.device.type == "cuda" else -1
    if rows.dim() != 2 or rows.shape != parents.shape or rows.dtype != torch.int32 or parents.dtype != torch.int32 \
            or not rows.get_device() == parents.get_device() == device:
        raise ValueError(f"rows and parents int32 [groups, beams] on {states.device}, not {rows.dtype} {tuple(rows.shape)} on {rows.device} and "
                         f"{parents.dtype} {tuple(parents.shape)} on {parents.device}")
    groups, beams = rows.shape
    if beams > MOST_BEAMS or groups > 65535:
        raise ValueError(f"{groups} groups of {beams} beams: up to 65535 of {MOST_BEAMS}")
    if lengths is not None and (not states.paged or lengths.shape != (groups,) or lengths.dtype != torch.int32 or lengths.get_device() != device):
        raise ValueError(f"lengths int32 [{groups}] on {states.device} for pages, not {lengths.dtype} {tuple(lengths.shape)} on {lengths.device}")
    if groups == 0 or beams == 0:
        return
    if device < 0:
        return ref.reorder_beams(states.tensors, rows, parents, lengths, states.int4_dim)
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return reorder_beams(states, rows, parents, lengths)
    stream = _native.stream_ptr()
    if stream != states._stream:
        states._table.record_stream(torch.cuda.current_stream())
    rows, parents = rows.contiguous(), parents.contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    rc = _native.lib().b200_beam_reorder(_REORDER.pack(
        states._table.data_ptr(), rows.data_ptr(), parents.data_ptr(), 0 if lengths is None else lengths.data_ptr(),
        _native.status_word(rows.device).data_ptr(), stream, len(states.tensors), groups, beams, states._wide,
        _native.sm_count(device)))
    _native.check(rc, "beam_reorder")
    wide = states._wide if beams <= 16 else 0
    _native.count_launch((wide > 0) + (wide < len(states.tensors)))
