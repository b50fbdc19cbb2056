"""Tensors whose rows lie between each other's: accepted where no byte is moved twice, refused where one is."""
import random

import pytest
import torch

from vllm_ascend_b200 import ops


def _bytes(t):
    """Elements of the buffer that a view holds."""
    at = torch.arange(t.untyped_storage().nbytes() // t.element_size())
    return set(at.as_strided(t.shape, t.stride(), t.storage_offset()).reshape(-1).tolist())


def _accepted(tensors, paged):
    try:
        ops.beam_states(tensors, paged=paged)
        return True
    except ValueError as e:
        assert "share memory" in str(e)
        return False


def test_rows_that_are_no_multiple_of_their_pieces_apart():
    buf = torch.zeros(700)
    a, b = (buf.as_strided((4, 2, 2, 5), (125, 5, 50, 1), first) for first in (0, 70))
    assert len(_bytes(a) & _bytes(b)) == 15
    with pytest.raises(ValueError, match="share memory"):
        ops.beam_states([a, b], paged=True)
    c = buf.as_strided((4, 2, 2, 5), (125, 5, 50, 1), 10)               # between the pieces of every row
    assert not _bytes(a) & _bytes(c)
    ops.beam_states([a, c], paged=True)


def test_pieces_of_padded_rows():
    each = torch.zeros(5 * (3 * 2 * 16 * 4 + 8))         # keys and values of a head side by side, eight elements behind every page
    k, v = (each.as_strided((5, 16, 3, 4), (392, 4, 128, 1), first) for first in (0, 64))
    assert not _bytes(k) & _bytes(v)
    ops.beam_states([k, v], paged=True)


@pytest.mark.parametrize("seed", range(8))
def test_pairs_of_pages(seed):
    """Pairs of one layout at any distance: what is accepted shares nothing, and what shares nothing is accepted."""
    rng = random.Random(seed)
    seen = set()
    for _ in range(150):
        heads, units, dim = rng.randint(1, 3), rng.randint(1, 3), rng.randint(1, 4)
        one = units * dim
        run = one + rng.choice([0, 0, one, rng.randint(0, 9)])
        row = (heads - 1) * run + one + rng.choice([0, run, rng.randint(0, 25)])
        n, n2 = rng.randint(1, 4), rng.randint(1, 4)
        first = rng.randint(0, 2 * row)
        buf = torch.zeros(7 * row + 100)
        a = buf.as_strided((n, units, heads, dim), (row, dim, run, 1), 0)
        b = buf.as_strided((n2, units, heads, dim), (row, dim, run, 1), first)
        apart = not _bytes(a) & _bytes(b)
        assert _accepted([a, b], True) == apart, (a.shape, a.stride(), b.shape, first)
        seen.add(apart)
    assert seen == {True, False}


@pytest.mark.parametrize("seed", range(4))
def test_rows_of_any_distance(seed):
    """Rows at other distances: what is accepted shares nothing."""
    rng = random.Random(seed)
    for _ in range(300):
        pair = []
        buf = torch.zeros(400)
        for _ in range(2):
            n, size = rng.randint(1, 5), rng.randint(1, 12)
            pair.append(buf.as_strided((n, size), (size + rng.randint(0, 30), 1), rng.randint(0, 60)))
        assert not (_accepted(pair, False) and _bytes(pair[0]) & _bytes(pair[1]))
