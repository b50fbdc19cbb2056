"""Calls of attention over a 4-bit cache that its other tests do not make: bad pages beside good ones, tables that are views, windows as wide
as their type, neighbours in modes with a fixed order of sums."""
import pytest
import torch

from test_gpu_kv_int4 import DEV, _check, _meta, _setup, _want, kernel  # noqa: F401
from vllm_ascend_b200 import _native, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("each", [1, 5])
def test_bad_pages_beside_good_ones(each):
    """A warp that meets a bad page ends; its neighbours wait for the copies that they have under way, and other sequences keep their bits."""
    lens = [2048 - 31 * i for i in range(48)]
    q, kc, vc, meta = _setup([each] * 48, lens, 16, 8, 2, 128, 40)
    good = ops.paged_attention_int4(q, kc, vc, meta, 0.1)
    table = meta.block_table.clone()
    for i in range(0, 48, 2):
        meta.block_table[i, (7 * i) % 36] = kc.shape[0] + i
        meta.block_table[i, 35] = -1
    for _ in range(5):
        out = ops.paged_attention_int4(q, kc, vc, meta, 0.1)
        with pytest.raises(_native.NativeError, match="BAD_INDEX"):
            _native.check_status(torch.device(DEV))
        rows = torch.arange(len(q), device=DEV) // each % 2 == 1
        assert torch.equal(out[rows], good[rows])
    meta.block_table.copy_(table)
    assert torch.equal(ops.paged_attention_int4(q, kc, vc, meta, 0.1), good)
    _native.check_status(torch.device(DEV))


@pytest.mark.parametrize("new", [[1, 1, 1], [1, 90, 130]])
def test_row_numbers_lengths_and_tables_that_are_views(new, kernel):
    """Every second or third element of larger tensors, as slices of a batch's columns are."""
    q, kc, vc, meta = _setup(new, [200, 333, 150], 32, 8, 2, 128, 41)
    want = ops.paged_attention_int4(q, kc, vc, meta, 0.1)
    _check(want, *_want(q, kc, vc, meta, 0.1))
    for name, step in (("query_start_loc", 2), ("seq_lens", 3), ("block_table", 2)):
        dense = getattr(meta, name)
        wide = torch.full((*dense.shape, step), 1 << 20, dtype=torch.int32, device=DEV)
        wide[..., 0] = dense
        setattr(meta, name, wide[..., 0])
        assert torch.equal(ops.paged_attention_int4(q, kc, vc, meta, 0.1), want), name
    _native.check_status(torch.device(DEV))
