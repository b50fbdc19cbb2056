"""Plans for lengths at the end of their type."""
import pytest
import torch

from shared_prefix_cases import Batch
from vllm_ascend_b200 import _native, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 100, 2 ** 31 - 127, 2 ** 31 - 128])
def test_the_longest_lengths_are_reported(length):
    b = Batch([(300, [(20, 1), (20, 1), (20, 1), (20, 1)])], 8, 8, 128, 128, device="cuda")
    b.meta.seq_lens.fill_(length)
    b.prefixes = torch.zeros_like(b.prefixes)
    out = torch.full((b.rows, 8, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    b.run(ops, out)
    torch.cuda.synchronize()
    with pytest.raises(_native.NativeError, match="BAD_INDEX"):
        _native.check_status(b.q.device)
    assert out.eq(3).all()
