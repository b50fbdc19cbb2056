"""Calls of the 4-bit cache's operators that its other tests on the host do not make."""
import dataclasses

import pytest
import torch

from test_kv_int4_cpu import _meta
from test_kv_int4_engine_cpu import _cfg
from vllm_ascend_b200 import ops


def test_caches_begin_on_16_bytes():
    """The kernels' bulk copies and wide stores need it, wherever the cache was cut from."""
    size = 2 * 2 * 16 * 64 * 9 // 16
    pool = torch.zeros(size + 64, dtype=torch.uint8)
    pool = pool[-pool.data_ptr() % 16:]
    whole, rows, slots = pool[:size].view(2, 2, -1), torch.zeros(1, 2, 64), torch.zeros(1, dtype=torch.int64)
    meta = _meta([1], [1], torch.zeros(1, 1, dtype=torch.int32), 4, 2, 64)
    ops.write_kv_int4(rows, rows, whole, whole.clone(), slots)
    for at in (1, 2, 4, 8):
        odd = pool[at:at + size].view(2, 2, -1)
        for pair in ((odd, whole), (whole, odd)):
            with pytest.raises(ValueError, match="16 bytes"):
                ops.write_kv_int4(rows, rows, *pair, slots)
            with pytest.raises(ValueError, match="16 bytes"):
                ops.read_kv_int4(*pair, slots, 64)
            with pytest.raises(ValueError, match="16 bytes"):
                ops.paged_attention_int4(torch.zeros(1, 4, 64), *pair, meta, 0.125)


def test_metadata_of_other_shapes_is_refused():
    kc, vc = (ops.alloc_kv_cache_int4(2, 16, 2, 64, "cpu") for _ in "kv")
    meta = _meta([1, 1], [1, 1], torch.zeros(2, 1, dtype=torch.int32), 4, 2, 64)
    for kw in (dict(block_table=meta.block_table[:, 0]), dict(seq_lens=meta.seq_lens.view(2, 1)), dict(query_start_loc=meta.query_start_loc.view(3, 1))):
        with pytest.raises(ValueError, match="metadata of 2 sequences"):
            ops.paged_attention_int4(torch.zeros(2, 4, 64), kc, vc, dataclasses.replace(meta, **kw), 0.125)


class _OnADevice:
    """A cache on a device whose copies to the host arrive when it is waited for: a copy that does not block holds zeros until then."""
    is_cuda, device = True, torch.device("cuda", 0)

    def __init__(self, data):
        self.data, self.dtype, self.shape = data, data.dtype, data.shape

    def dim(self):
        return self.data.dim()

    def __getitem__(self, at):
        return _OnADevice(self.data[at])

    def to(self, device, non_blocking=False):
        assert torch.device(device).type == "cpu"
        return torch.zeros_like(self.data) if non_blocking else self.data.clone()


def test_swapped_blocks_have_arrived_on_the_host(monkeypatch):
    from vllm_ascend_b200.attention.backend import B200AttentionBackend
    host, pairs, to = ops.alloc_kv_cache_int4(3, 16, 2, 64, "cpu"), torch.tensor([[0, 2], [3, 1]]), torch.Tensor.to
    src = torch.randint(1, 255, (4, *host.shape[1:]), dtype=torch.uint8)
    monkeypatch.setattr(torch.Tensor, "to", lambda t, d, *a, **kw: t if torch.device(d).type == "cuda" else to(t, d, *a, **kw))     # the pairs
    B200AttentionBackend.swap_blocks(_OnADevice(src), host, pairs)
    assert torch.equal(host[2], src[0]) and torch.equal(host[1], src[3]) and not host[0].any()


@pytest.mark.parametrize("causal,window", [(True, 0), (True, 9), (False, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_is_no_number_reaches_the_rows_that_see_it(causal, window, dtype):
    """A group of keys takes a row's heads of the group whole, one of values its 32 channels; other rows have the bits they have without it."""
    g = torch.Generator().manual_seed(window)
    Hq, Hkv, D, page, new, lens = 6, 2, 64, 16, [1, 6, 3], [30, 21, 48]
    table = torch.tensor([[5, 1, 0], [2, 7, 0], [3, 4, 6]], dtype=torch.int32)
    kc, vc = (ops.alloc_kv_cache_int4(8, page, Hkv, D, "cpu") for _ in "kv")
    k, v = (torch.randn(8 * page, Hkv, D, generator=g).to(dtype) for _ in "kv")
    ops.write_kv_int4(k, v, kc, vc, torch.arange(8 * page))
    q, meta = torch.randn(sum(new), Hq, D, generator=g).to(dtype), _meta(new, lens, table, Hq, Hkv, D)
    spots = [(0, 28, "v"), (0, 31, "v"), (1, 17, "k"), (1, 19, "v"), (1, 25, "k"), (2, 2, "k"), (2, 46, "v"), (2, 47, "k")]
    slots = torch.stack([table[b, t // page].long() * page + t % page for b, t, _ in spots])
    want = ops.paged_attention_int4(q, kc, vc, meta, 0.125, causal=causal, window=window)
    assert torch.isfinite(want).all()
    hit = torch.zeros_like(want, dtype=torch.bool)
    for i, (b, t, what) in enumerate(spots):
        (k if what == "k" else v)[slots[i], 1 if what == "k" else 0, 40] = float("inf" if i % 2 else "nan")
        for row, pos in enumerate(range(lens[b] - new[b], lens[b]), sum(new[:b])):
            if t >= lens[b] or causal and t > pos or window and t <= pos - window:
                continue
            hit[row, slice(3, 6) if what == "k" else slice(0, 3), 0 if what == "k" else 32:] = True
    ops.write_kv_int4(k, v, kc, vc, torch.arange(8 * page))
    out = ops.paged_attention_int4(q, kc, vc, meta, 0.125, causal=causal, window=window)
    assert out.isnan().equal(hit) and torch.equal(out[~hit], want[~hit])


@pytest.mark.parametrize("method,layers", [("eagle", 1), ("eagle3", 1), ("draft_model", 3), ("ngram", 0)])
@pytest.mark.parametrize("kv", ["int4", "auto"])
def test_draft_caches_count_against_the_memory_of_blocks(method, layers, kv, monkeypatch):
    """Drafts keep keys and values of every block in the model's type, whatever the model's own cache is."""
    from vllm_ascend_b200.engine.llm import LLM
    from vllm_ascend_b200.engine.model_runner import ModelRunner
    from vllm_ascend_b200.engine.request import SamplingParams
    made, whole = [], ModelRunner.determine_num_blocks
    monkeypatch.setattr(ModelRunner, "determine_num_blocks", lambda r: made.append(r.proposer) or whole(r))
    spec = {"method": method, "num_speculative_tokens": 2, "model": _cfg(name="d", num_hidden_layers=3, num_key_value_heads=4, dtype="bfloat16")}
    llm = LLM(_cfg(dtype="bfloat16"), device="cpu", max_model_len=1 << 16, max_num_seqs=2, block_size=16, max_num_batched_tokens=64, kv_cache_dtype=kv,
              num_gpu_blocks_override=64, speculative_config={k: v for k, v in spec.items() if k != "model" or method == "draft_model"})
    r = llm.engine.runner
    assert made == [r.proposer]                                    # its weights are there when the rest is measured
    heads = 4 if method == "draft_model" else 2
    draft = layers * 2 * 16 * heads * 64 * 2
    assert r.draft_bytes_per_block() == draft
    llm.generate([[3, 4, 5] * 9], SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True))
    if layers:
        assert sum(t[0].numel() * t.element_size() for c in r.proposer.kv_caches for t in c) == draft
    room = 100 * (r.kv_bytes_per_block() + draft) + 5
    r.is_cuda, r.cfg.cache.num_gpu_blocks = True, None
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(r, "activation_bytes_estimate", lambda: 0)
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda *a: (room, room))
    r.cfg.cache.gpu_memory_utilization = 1.0
    assert r.determine_num_blocks() == 100


def test_names_of_cache_types(caplog):
    """Text that names no type is refused; types that there is no cache of are stored in the model's, with a word."""
    import logging
    from vllm_ascend_b200.config import CacheConfig
    from vllm_ascend_b200.engine.llm import LLM
    small = dict(device="cpu", max_model_len=64, max_num_seqs=2, block_size=16)
    for text in ("INT4", "int4 ", "int-4", "", "4"):
        with pytest.raises(ValueError, match="kv_cache_dtype"):
            LLM(_cfg(), kv_cache_dtype=text, **small)
    assert CacheConfig(kv_cache_dtype=None).kv_cache_dtype == "auto"
    logger = logging.getLogger("vllm_ascend_b200")
    logger.addHandler(caplog.handler)
    try:
        for text, said in (("auto", False), ("float32", False), ("int4", False), ("fp8", True), ("bfloat16", True)):
            caplog.clear()
            caches = LLM(_cfg(), kv_cache_dtype=text, **small).engine.runner.kv_caches
            assert caches[0][0].dtype is (torch.uint8 if text == "int4" else torch.float32)
            assert any("kv_cache_dtype" in r.getMessage() for r in caplog.records) is said
    finally:
        logger.removeHandler(caplog.handler)
