"""The largest vocabularies that a selection takes: positions count past a row's end in 32 bits."""
import pytest
import torch

from vllm_ascend_b200 import _native, ops
from vllm_ascend_b200.ops import beam

TILE = 4096


def _guard(vocab, parts, per):
    """What the launcher says to one row of so many tokens; it launches nothing here."""
    return _native.lib().b200_beam_select(beam._SELECT.pack(*([0] * 11), vocab, 1, 1, vocab, 1, parts, per, 0, 0))


@pytest.mark.skipif(torch.cuda.is_available(), reason="sizes in range would launch")
def test_positions_past_the_end_stay_below_31_bits():
    last = 2 ** 31 - 1 - 8 * TILE                        # a walk looks that far past a row
    for vocab in (last + 1, 2 ** 31 - 1 - 3 * TILE, 2 ** 31 - 1):
        tiles = -(-(vocab + 7) // TILE)
        for parts in (1, 2, 17, 148):
            per = -(-tiles // parts) * TILE
            assert _guard(vocab, parts, min(per, 2 ** 31 - TILE)) in (9931, 9932)
    tiles = -(-(last - 7) // TILE)
    assert _guard(last - 7, 1, tiles * TILE) not in (9930, 9931, 9932, 9933)         # in range: what a machine without a GPU answers
    assert _guard(1000, 5, TILE) == 9932                 # parts behind the last element


def test_vocabularies_that_are_refused():
    for vocab in (2 ** 31 - 1, 2 ** 31 - 1 - 8 * TILE + 1):
        with pytest.raises(ValueError, match="tokens"):
            ops.beam_select(torch.empty((1, vocab), device="meta"), torch.zeros((1, 1), device="meta"), 1)
