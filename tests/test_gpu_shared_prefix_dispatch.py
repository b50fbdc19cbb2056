"""Attention with a plan for shared prefixes in its metadata, where the kernel for it does not take the sizes."""
import pytest
import torch

from shared_prefix_cases import Batch
from vllm_ascend_b200 import ops
from vllm_ascend_b200.ops import shared_prefix

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim,page", [(torch.bfloat16, 64, 24), (torch.bfloat16, 64, 16), (torch.float32, 128, 16), (torch.bfloat16, 40, 16)])
def test_plans_without_a_kernel_are_not_followed(monkeypatch, dtype, dim, page):
    b = Batch([(480, [(20, 1), (33, 1), (7, 1)])], 8, 2, dim, page, device="cuda", dtype=dtype, order="tokens")
    whole = 480 // page
    b.meta.block_table[:, :whole] = b.meta.block_table[:1, :whole].clone()              # rows that hold whole sequences
    b.meta.block_table[b.meta.block_table >= 10 ** 6] = 0
    for cache in (b.k_cache, b.v_cache):
        cache[cache.isnan()] = 0
    want = ops.paged_attention(b.q.contiguous(), b.k_cache, b.v_cache, b.meta, b.scale)
    b.check(want)
    b.meta.shared = b.plan(ops)
    monkeypatch.setattr(shared_prefix, "_definition", lambda *a: pytest.fail("a loop over sequences"))
    calls = []
    monkeypatch.setattr(ops, "paged_attention_shared", lambda *a: calls.append(1) or shared_prefix.paged_attention_shared(*a))
    got = ops.paged_attention(b.q.contiguous(), b.k_cache, b.v_cache, b.meta, b.scale)
    b.check(got)
    assert bool(calls) == shared_prefix.has_kernel(dtype, dim, page) and (calls or torch.equal(got, want))
