"""The engine with its cache in 4 bits (``kv_cache_dtype="int4"``): what it generates, how much it stores, what it refuses."""
import numpy as np
import pytest
import torch

from vllm_ascend_b200 import ops
from vllm_ascend_b200.attention.metadata import AttentionMetadata
from vllm_ascend_b200.config import ModelConfig, get_model_config
from vllm_ascend_b200.engine.llm import LLM
from vllm_ascend_b200.engine.request import SamplingParams


def _cfg(**kw):
    return ModelConfig(**{**dict(name="t", architecture="Qwen3ForCausalLM", vocab_size=256, hidden_size=128, intermediate_size=192,
                                 num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64, qk_norm=True,
                                 rope_theta=1e6, dtype="float32", init_std=0.08), **kw})


def _greedy(llm, prompt, n, page=16):
    """Tokens of a model that sees its whole sequence at once, over a fresh 4-bit cache every time."""
    model, ids = llm.engine.runner.model, list(prompt)
    for _ in range(n):
        T = len(ids)
        blocks = -(-T // page) + 1
        caches = [tuple(ops.alloc_kv_cache_int4(blocks, page, L.self_attn.Hkv, L.self_attn.D, "cpu") for _ in "kv") for L in model.layers]
        pos = torch.arange(T)
        meta = AttentionMetadata(
            num_reqs=1, num_actual_tokens=T, max_query_len=T, max_seq_len=T, query_start_loc=torch.tensor([0, T], dtype=torch.int32),
            seq_lens=torch.tensor([T], dtype=torch.int32), block_table=torch.arange(1, blocks, dtype=torch.int32).unsqueeze(0),
            slot_mapping=pos + page, positions=pos, query_start_loc_cpu=np.array([0, T]), seq_lens_cpu=np.array([T]))
        with torch.no_grad():
            h = model.forward(torch.tensor(ids), meta, caches)
            ids.append(int(model.compute_logits(h[-1:]).argmax()))
    return ids[len(prompt):]


@pytest.mark.parametrize("kw", [{}, {"enable_prefix_caching": True}, {"max_num_batched_tokens": 32},
                                {"speculative_config": {"method": "ngram", "num_speculative_tokens": 2}}])
def test_generation_over_a_4_bit_cache(kw):
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, 256, size=n).tolist() for n in (5, 40, 17)]
    prompts.append(prompts[1][:32] + [3, 4, 5])
    llm = LLM(_cfg(), device="cpu", max_model_len=128, max_num_seqs=4, block_size=16, kv_cache_dtype="int4", **kw)
    caches = llm.engine.runner.kv_caches
    assert all(t.dtype == torch.uint8 and t.shape[1:] == (2, 16 * 64 * 9 // 16) for pair in caches for t in pair)
    outs = llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True))
    for p, o in zip(prompts, outs):
        assert o.outputs[0].token_ids == _greedy(llm, p, 6)


def test_blocks_take_9_bits_of_32():
    full = LLM(_cfg(), device="cpu", max_model_len=64, max_num_seqs=2, block_size=16).engine.runner
    four = LLM(_cfg(), device="cpu", max_model_len=64, max_num_seqs=2, block_size=16, kv_cache_dtype="int4").engine.runner
    assert four.kv_bytes_per_block() * 64 == full.kv_bytes_per_block() * 9           # fp32 here: 4.5 bits instead of 32
    assert four.kv_bytes_per_block() == sum(t[0].numel() for pair in four.kv_caches for t in pair)


def test_refusals():
    small = dict(device="cpu", max_model_len=64, max_num_seqs=2, block_size=16, kv_cache_dtype="int4")
    with pytest.raises(ValueError, match="takes heads"):
        LLM(_cfg(head_dim=32), **small)
    with pytest.raises(ValueError, match="takes blocks"):
        LLM(_cfg(), **{**small, "block_size": 8})
    with pytest.raises(NotImplementedError, match="latent"):
        LLM(get_model_config("tiny-deepseek"), **small)
    with pytest.raises(NotImplementedError, match="plan-built"):
        LLM(get_model_config("tiny-nevotar"), **small)
    runner = LLM(_cfg(), **small).engine.runner
    runner.is_cuda = True                        # float32: its rows would go through the host's definitions, which no graph can hold
    with pytest.raises(NotImplementedError, match="float32 on a GPU"):
        runner.kv_bytes_per_block()


def test_dispatcher_schema_and_copied_blocks():
    import vllm_ascend_b200.ops.torch_bindings as tb
    from vllm_ascend_b200.attention.backend import B200AttentionBackend
    from vllm_ascend_b200.attention.metadata import metadata_from_tensors
    tb.register()
    g = torch.Generator().manual_seed(5)
    kc, vc = (ops.alloc_kv_cache_int4(4, 16, 2, 64, "cpu") for _ in "kv")
    ops.write_kv_int4(*(torch.randn(32, 2, 64, generator=g) for _ in "kv"), kc, vc, torch.arange(32))
    q = torch.randn(3, 4, 64, generator=g)
    cu, lens = torch.tensor([0, 1, 3], dtype=torch.int32), torch.tensor([16, 9], dtype=torch.int32)
    table = torch.tensor([[0], [1]], dtype=torch.int32)
    out = ops.paged_attention(q, kc, vc, metadata_from_tensors(cu, lens, table, 2, 16, 4, 2, 64), 0.125)
    assert torch.equal(getattr(torch.ops, tb.NAMESPACE).paged_attention(q, kc, vc, table, lens, cu, 2, 16, 0.125, True, 0), out)
    B200AttentionBackend.copy_blocks([(kc, vc)], torch.tensor([[0, 3], [1, 2]]))
    moved = metadata_from_tensors(cu, lens, 3 - table, 2, 16, 4, 2, 64)
    assert torch.equal(ops.paged_attention(q, kc, vc, moved, 0.125), out)
