"""Selection over beams and vocabulary and reordering of states: definitions on the host, refusals."""
import math

import pytest
import torch

from beam_cases import check_select, reorder
from vllm_ascend_b200 import ops


def test_definition_of_the_selection():
    g = torch.Generator().manual_seed(0)
    logits, scores = torch.randn(12, 301, generator=g), -torch.rand(3, 4, generator=g)
    logits[1, 5], logits[2] = math.nan, -math.inf
    scores[1, 1] = -math.inf
    for x in (logits, logits.bfloat16(), logits.half(), logits.double()):
        check_select(ops.beam_select(x, scores, 9), x, scores, 9)
    assert ops.beam_select(logits, scores)[0].shape == (3, 8)
    assert ops.beam_select(logits[:, :1], scores)[0].shape == (3, 4)


@pytest.mark.parametrize("logits,scores,k", [
    (torch.zeros(6), torch.zeros(2, 3), 2), (torch.zeros(6, 5), torch.zeros(6), 2), (torch.zeros(5, 5), torch.zeros(2, 3), 2),
    (torch.zeros(6, 5), torch.zeros(2, 3).double(), 2), (torch.zeros(6, 5).long(), torch.zeros(2, 3), 2), (torch.zeros(6, 5), torch.zeros(2, 3), 0),
    (torch.zeros(6, 5), torch.zeros(2, 3), 16), (torch.zeros(6, 500), torch.zeros(2, 3), 257), (torch.zeros(0, 5), torch.zeros(2, 0), 1),
    (torch.zeros(6, 0), torch.zeros(2, 3), 1), (torch.zeros(1025, 3), torch.zeros(1, 1025), 4)])
def test_selections_that_are_refused(logits, scores, k):
    with pytest.raises(ValueError):
        ops.beam_select(logits, scores, k)


def test_definition_of_the_reordering():
    g = torch.Generator().manual_seed(1)
    tensors = [torch.randn(9, 4, generator=g), torch.randint(0, 9, (9, 2, 3), generator=g)]
    rows, parents = torch.tensor([[8, 1, 4], [0, 2, -1]], dtype=torch.int32), torch.tensor([[1, 2, 0], [1, -1, 0]], dtype=torch.int32)
    want = reorder(tensors, rows, parents)
    ops.reorder_beams(ops.beam_states(tensors), rows, parents)
    assert all(torch.equal(a, b) for a, b in zip(tensors, want))
    pages = [torch.randn(9, 16, 2, 4, generator=g), torch.randn(9, 2, 16, 4, generator=g).transpose(1, 2)]
    lengths = torch.tensor([3, 0], dtype=torch.int32)
    want = reorder(pages, rows, parents, lengths)
    ops.reorder_beams(ops.beam_states(pages, paged=True), rows, parents, lengths)
    assert all(torch.equal(a, b) for a, b in zip(pages, want))


def test_reorderings_that_are_refused():
    x, rows = torch.zeros(6, 16, 2, 4), torch.zeros((1, 3), dtype=torch.int32)
    for tensors, paged in (([], False), ([torch.zeros(6, 4, 5).transpose(1, 2)], False), ([torch.zeros(6, 4)], True),
                           ([torch.zeros(1, 4).expand(6, 4)], False), ([torch.zeros(6, 2, 4, 16).permute(0, 3, 1, 2)], True),
                           ([torch.zeros(6, 2, 4, 16).permute(0, 2, 3, 1)], True), ([torch.zeros((6, 2, 100), dtype=torch.uint8)], True)):
        with pytest.raises(ValueError):
            ops.beam_states(tensors, paged=paged)
    with pytest.raises(ValueError):
        ops.beam_states([torch.zeros((6, 2, 577), dtype=torch.uint8)], paged=True, int4_dim=64)
    plain, pages = ops.beam_states([x]), ops.beam_states([x], paged=True)
    for states, r, p, n in ((plain, rows.long(), rows, None), (plain, rows, rows[:, :2], None), (plain, rows[0], rows[0], None),
                            (plain, rows, rows, torch.zeros(1, dtype=torch.int32)), (pages, rows, rows, torch.zeros(2, dtype=torch.int32)),
                            (pages, rows, rows, torch.zeros(1)), (plain, torch.zeros((1, 1025), dtype=torch.int32),
                                                                  torch.zeros((1, 1025), dtype=torch.int32), None)):
        with pytest.raises(ValueError):
            ops.reorder_beams(states, r, p, n)
    for r, p in (([[0, 1, 6]], [[0, 0, 0]]), ([[0, 1, 2]], [[0, 3, 0]]), ([[0, -1, 2]], [[1, 0, 0]])):
        with pytest.raises(IndexError):
            ops.reorder_beams(plain, torch.tensor(r, dtype=torch.int32), torch.tensor(p, dtype=torch.int32))


def test_tensors_that_share_memory_are_refused():
    x, slices = torch.zeros(6, 16, 2, 4), torch.arange(6 * 12.).view(6, 12)
    for tensors, paged in (([x, x], False), ([x, x[2:]], False), ([x.view(6, -1)[:, :100], x.view(6, -1)[:, 96:]], False), ([x, x], True),
                           ([slices, slices.view(12, 6)], False), ([slices[:, :4], slices[:, 8:], slices[2:, 2:6]], False)):
        with pytest.raises(ValueError, match="share memory"):
            ops.beam_states(tensors, paged=paged)
    both = torch.zeros(5, 2, 3, 16, 4)                   # keys and values of a page side by side
    ops.beam_states([both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)], paged=True)
    each = torch.zeros(5, 3, 2, 16, 4)                   # of a head
    ops.beam_states([each[:, :, 0].transpose(1, 2), each[:, :, 1].transpose(1, 2)], paged=True)
    ops.beam_states([slices[:3], slices[3:]])
    parts = [slices[:, :4], slices[:, 4:]]
    rows, parents = torch.tensor([[0, 5]], dtype=torch.int32), torch.tensor([[1, 0]], dtype=torch.int32)
    want = slices[[5, 1, 2, 3, 4, 0]]
    ops.reorder_beams(ops.beam_states(parts), rows, parents)
    assert torch.equal(slices, want)
