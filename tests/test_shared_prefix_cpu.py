"""Attention of batches that share prefixes: definition on the host, refusals."""
import pytest
import torch

from shared_prefix_cases import Batch
from vllm_ascend_b200 import ops


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_definition(dtype, order):
    b = Batch([(21, [(5, 1), (9, 2), (1, 1)]), (0, [(4, 1)]), (16, [(3, 3), (20, 1)])], 4, 2, 8, 8, alone=[(7, 1)], dtype=dtype, order=order)
    b.check(b.run(ops))


def test_prefixes_end_in_front_of_new_tokens():
    b = Batch([(16, [(4, 2), (4, 2)])], 4, 2, 8, 8, dtype=torch.float32)
    b.prefixes += 50                                    # reaches into what differs: counts up to 18
    table = b.meta.block_table
    table[1, 2] = table[0, 2]
    b.keys[1][16:18], b.values[1][16:18] = b.keys[0][16:18], b.values[0][16:18]
    page = int(table[0, 2])
    for cache, rows in ((b.k_cache, b.keys), (b.v_cache, b.values)):
        other = int(b.table[1, 2])
        assert other == page
    b.keys[1], b.values[1] = b.keys[0], b.values[0]
    b.check(b.run(ops))


def test_paged_attention_agrees():
    b = Batch([(16, [(5, 1), (9, 2)])], 4, 2, 8, 8, dtype=torch.float32)
    whole = Batch([(0, [(21, 1)]), (0, [(25, 2)])], 4, 2, 8, 8, dtype=torch.float32)
    whole.keys, whole.values, whole.q = b.keys, b.values, b.q
    for s, (k, v) in enumerate(zip(b.keys, b.values)):
        for pos in range(len(k)):
            whole.k_cache[int(whole.table[s, pos // 8]), pos % 8], whole.v_cache[int(whole.table[s, pos // 8]), pos % 8] = k[pos], v[pos]
    a = ops.paged_attention(whole.q.contiguous(), whole.k_cache, whole.v_cache, whole.meta, whole.scale)
    assert torch.allclose(a, b.run(ops), atol=1e-5)


def test_refusals():
    b = Batch([(16, [(5, 1), (9, 2)])], 4, 2, 8, 8, dtype=torch.float32)
    plan = b.plan(ops)
    for starts, prefixes, heads, kv in ((b.starts.long(), b.prefixes, 4, 2), (b.starts, b.prefixes[:0], 4, 2), (b.starts, b.prefixes, 4, 3),
                                        (b.starts, b.prefixes, 129, 1), (b.starts[None], b.prefixes, 4, 2), (b.starts, b.prefixes, 4, 0)):
        with pytest.raises(ValueError):
            ops.plan_shared_prefix(b.meta, starts, prefixes, heads, kv)
    q, k, v = b.q, b.k_cache, b.v_cache
    for args in ((q[0], k, v, b.meta, plan, 1.0), (q[:, :2], k, v, b.meta, plan, 1.0), (q.half(), k, v, b.meta, plan, 1.0),
                 (q, k, v[:, :4], b.meta, plan, 1.0), (q, k, v, b.meta, plan, 0.0), (q, k, v, b.meta, plan, float("nan")),
                 (q, k, v, b.meta, plan, 1.0, torch.empty(3, 4, 7)), (q[:2], k, v, b.meta, plan, 1.0), (q[..., :4], k, v, b.meta, plan, 1.0)):
        with pytest.raises(ValueError):
            ops.paged_attention_shared(*args)
    with pytest.raises(IndexError):
        bad = ops.plan_shared_prefix(b.meta, torch.tensor([1, 0], dtype=torch.int32), b.prefixes, 4, 2)
        ops.paged_attention_shared(q, k, v, b.meta, bad, 1.0)


def test_a_plan_is_not_used_for_another_batch():
    import copy
    b = Batch([(16, [(5, 1), (9, 1)])], 4, 2, 8, 8, dtype=torch.float32)
    meta = b.meta
    meta.block_table[1, :2] = meta.block_table[0, :2]
    meta.shared = b.plan(ops)
    want = b.run(ops)
    assert torch.equal(ops.paged_attention(b.q.contiguous(), b.k_cache, b.v_cache, meta, b.scale), want)
    other = copy.copy(meta)                              # what a drafter does with a step's metadata
    other.seq_lens, other.seq_lens_cpu = meta.seq_lens - 1, meta.seq_lens_cpu - 1
    got = ops.paged_attention(b.q.contiguous(), b.k_cache, b.v_cache, other, b.scale)
    other.shared = None
    assert torch.equal(got, ops.paged_attention(b.q.contiguous(), b.k_cache, b.v_cache, other, b.scale))
    assert not torch.allclose(got, want)
