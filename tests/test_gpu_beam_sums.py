"""Sums of exponentials whose terms lie far below a row's largest element, to more bits than a 32-bit exponential of their distance has."""
import math

import pytest
import torch

from vllm_ascend_b200 import ops

pytestmark = pytest.mark.gpu

VOCAB = 151936
#: elements of a thread's share of a row, steps that it adds them in
SHARE, STEPS = 8 * 38, 38


def _worst(lo, hi):
    """The distance in fp32 for which the product with log2 e, rounded to fp32, is furthest from the exact one."""
    d = torch.linspace(lo, hi, 200001, dtype=torch.float32)
    off = (d * torch.tensor(math.log2(math.e), dtype=torch.float32)).double() - d.double() * math.log2(math.e)
    return float(d[off.abs().argmax()])


@pytest.mark.parametrize("lo,hi", [(2.0, 4.0), (5.6, 6.4), (8.0, 8.3)])
@pytest.mark.parametrize("rows", [2, 150])
def test_a_peak_over_a_flat_row(rows, lo, hi):
    """Beam 0: one element at 0, the others d below; beam 1: all elements equal, whose sum is a whole number.  A thread without the peak adds ones, which
    is exact.  The thread with it adds up to 1 + SHARE e^-d: half a step for every STEP, and its small terms are off by 2^-22 of their exponential
    and 2^-23 d of their distance.  Totals of the beams that are twice that apart come in their order."""
    d = _worst(lo, hi)
    logits = torch.full((rows, VOCAB), 0.25, dtype=torch.float32, device="cuda")
    logits[::2] = -d
    at = torch.randint(0, VOCAB, (rows // 2,), generator=torch.Generator().manual_seed(rows)).cuda()
    logits[torch.arange(0, rows, 2, device="cuda"), at] = 0.0
    total, small = 1 + (VOCAB - 1) * math.exp(-d), SHARE * math.exp(-d)
    off = (STEPS * 2.0 ** -24 * (1 + small) + small * (2.0 ** -22 + d * 2.0 ** -23)) / total + 1e-12
    peak = -math.log(total)
    values, _, tokens = ops.beam_select(logits[::2], torch.zeros((rows // 2, 1), dtype=torch.float64, device="cuda"), 1, dtype=torch.float64)
    assert torch.equal(tokens[:, 0], at)
    assert ((values - peak).abs() <= off).all(), float((values - peak).abs().max()) / off
    for gap in (2 * off, -2 * off):
        scores = torch.zeros((rows // 2, 2), dtype=torch.float64, device="cuda")
        scores[:, 1] = peak + math.log(VOCAB) + gap
        assert ops.beam_select(logits, scores, 1, dtype=torch.float64)[1].eq(1 if gap > 0 else 0).all()
