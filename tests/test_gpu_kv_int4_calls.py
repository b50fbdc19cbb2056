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


@pytest.mark.parametrize("new", [[1, 1, 1], [1, 90, 130]])
def test_tables_that_rows_share_or_that_are_cut_from_wider_ones(new, kernel):
    """One row of pages for all sequences (a row stride of zero); columns out of a table whose other entries are no pages, up to its very end."""
    lens = [200, 333, 150]
    q, kc, vc, meta = _setup(new, lens, 32, 8, 2, 128, 42)
    table = meta.block_table
    meta.block_table = table[1:2].expand(3, -1)
    out = ops.paged_attention_int4(q, kc, vc, meta, 0.1)
    _check(out, *_want(q, kc, vc, meta, 0.1))
    meta.block_table = table[1:2].repeat(3, 1)
    assert torch.equal(ops.paged_attention_int4(q, kc, vc, meta, 0.1), out)
    wide = torch.full((3, 40), 1 << 20, dtype=torch.int32, device=DEV)
    wide[:, 40 - table.shape[1]:] = table
    meta.block_table = table
    out = ops.paged_attention_int4(q, kc, vc, meta, 0.1)
    meta.block_table = wide[:, 40 - table.shape[1]:]
    assert torch.equal(ops.paged_attention_int4(q, kc, vc, meta, 0.1), out)
    _native.check_status(torch.device(DEV))


def test_lengths_beyond_the_columns_are_reported(kernel):
    """A sequence with more keys than its row of the table has pages: what lies behind the row is not read."""
    q, kc, vc, meta = _setup([1, 64], [333, 320], 32, 8, 2, 128, 43)
    wide = torch.zeros((2, 40), dtype=torch.int32, device=DEV)
    wide[:, :11] = meta.block_table
    meta.block_table = wide[:, :10]
    good = ops.paged_attention_int4(q, kc, vc, meta, 0.1)
    with pytest.raises(_native.NativeError, match="BAD_INDEX"):
        _native.check_status(torch.device(DEV))
    _check(good[1:], *(t[1:] for t in _want(q, kc, vc, _meta([1, 64], [320, 320], meta.block_table, 8, 2, 128), 0.1)))


@pytest.mark.parametrize("page,columns", [(128, 8192), (16, 70000), (256, 1 << 19)])
def test_tables_of_a_million_tokens_and_more(page, columns, kernel):
    """What a table could hold is no reason to refuse short sequences in it."""
    q, kc, vc, meta = _setup([1, 70], [300, 170], page, 8, 2, 128, 44)
    out = ops.paged_attention_int4(q, kc, vc, meta, 0.1)
    wide = torch.full((2, columns), -1, dtype=torch.int32, device=DEV)
    wide[:, :meta.block_table.shape[1]] = meta.block_table
    meta.block_table = wide
    assert torch.equal(ops.paged_attention_int4(q, kc, vc, meta, 0.1), out)
    _native.check_status(torch.device(DEV))


@pytest.mark.parametrize("new,lens,Hq,Hkv,window", [
    ([1, 1, 3], [1000, 3000, 700], 16, 2, 527), ([2, 3, 1], [900, 999, 40], 8, 2, 100), ([1, 4, 1, 1], [2049, 555, 2050, 2063], 8, 1, 1030)])
@pytest.mark.parametrize("D", [64, 128])
def test_fixed_sums_in_windows_beside_longer_neighbours(new, lens, Hq, Hkv, window, D, monkeypatch):
    """Eight rows of a sequence fill a tile alone; beside a neighbour of more rows, eight that do not exist join them in their block."""
    q, kc, vc, meta = _setup(new, lens, 32, Hq, Hkv, D, 45)
    monkeypatch.setattr("vllm_ascend_b200.ops.kv_int4.fixed_sums", lambda: True)
    out = ops.paged_attention_int4(q, kc, vc, meta, 0.1, window=window)
    _check(out, *_want(q, kc, vc, meta, 0.1, window))
    cu = meta.query_start_loc_cpu
    for b in range(len(new)):
        one = _meta(new[b:b + 1], lens[b:b + 1], meta.block_table[b:b + 1], Hq, Hkv, D)
        assert torch.equal(ops.paged_attention_int4(q[cu[b]:cu[b + 1]], kc, vc, one, 0.1, window=window), out[cu[b]:cu[b + 1]]), b


@pytest.mark.parametrize("window", [2 ** 31 - 2, 2 ** 31 - 1, 1 << 40])
def test_windows_wider_than_any_sequence(window, kernel):
    """The same as none, in front of the first key too, where positions are below zero."""
    q, kc, vc, meta = _setup([300, 3, 64, 1], [20, 1, 64, 500], 16, 8, 2, 128, 46)
    out = ops.paged_attention_int4(q, kc, vc, meta, 0.1, window=window)
    _check(out, *_want(q, kc, vc, meta, 0.1, window))
    assert torch.equal(ops.paged_attention_int4(q, kc, vc, meta, 0.1), out)


@pytest.mark.parametrize("pinned", [True, False])
def test_blocks_swapped_to_the_host_and_back(pinned):
    """A cache's blocks are on the host when the call returns, behind whatever work the device still had."""
    from vllm_ascend_b200.attention.backend import B200AttentionBackend
    g = torch.Generator().manual_seed(47)
    data = torch.randint(1, 255, (64, 8, 128 * 128 * 9 // 16), generator=g, dtype=torch.uint8)
    src, host = torch.zeros_like(data, device=DEV), torch.zeros(16, *data.shape[1:], dtype=torch.uint8, pin_memory=pinned)
    pairs = torch.tensor([[i * 5 % 64, i] for i in range(16)])
    big = torch.randn(8192, 8192, device=DEV, dtype=torch.bfloat16)
    for _ in range(3):
        for _ in range(20):
            big @ big
        src.copy_(data.to(DEV))
        B200AttentionBackend.swap_blocks(src, host, pairs)
        assert torch.equal(host, data[pairs[:, 0]])
        back = torch.zeros_like(src)
        B200AttentionBackend.swap_blocks(host, back, pairs.flip(1))
        assert torch.equal(back[pairs[:, 0].to(DEV)], src[pairs[:, 0].to(DEV)])
        host.zero_()
        src.zero_()


def test_slots_and_pages_out_of_range_with_other_types():
    """fp32 rows go through the operators' definition; what is out of range is reported as the kernels report it, the rest is done."""
    q, kc, vc, meta = _setup([1, 3], [50, 90], 16, 8, 2, 64, 48)
    want, tol = _want(q, kc, vc, meta, 0.2)
    k4, v4 = kc.clone(), vc.clone()
    rows = torch.ones(4, 2, 64, device=DEV)
    ops.write_kv_int4(rows, rows, k4, v4, torch.tensor([3, kc.shape[0] * 16, -1, 1 << 40], device=DEV))
    with pytest.raises(_native.NativeError, match="BAD_INDEX"):
        _native.check_status(torch.device(DEV))
    ops.write_kv_int4(rows[:1], rows[:1], kc, vc, torch.tensor([3], device=DEV))
    assert torch.equal(k4, kc) and torch.equal(v4, vc)
    want, tol = _want(q, kc, vc, meta, 0.2)
    for bad in (kc.shape[0], 1 << 30, -1, -(1 << 30)):
        page = int(meta.block_table[0, 2])
        meta.block_table[0, 2] = bad
        out = ops.paged_attention_int4(q.float(), kc, vc, meta, 0.2)
        with pytest.raises(_native.NativeError, match="BAD_INDEX"):
            _native.check_status(torch.device(DEV))
        assert float((out[1:].double() - want[1:]).abs().max()) < 1e-4
        meta.block_table[0, 2] = page
    # in front of a window, and behind a sequence's end, a table may hold anything
    for window in (1, 20):
        want, tol = _want(q, kc, vc, meta, 0.2, window)
        table = meta.block_table.clone()
        for b, n, a in ((0, 50, 1), (1, 90, 3)):
            meta.block_table[b, :max(0, n - a - window + 1) // 16] = -(1 << 30)
        out = ops.paged_attention_int4(q.float(), kc, vc, meta, 0.2, window=window)
        assert float((out.double() - want).abs().max()) < 1e-4
        _check(ops.paged_attention_int4(q, kc, vc, meta, 0.2, window=window), want, tol)
        meta.block_table.copy_(table)
    _native.check_status(torch.device(DEV))


def test_what_is_no_number_with_other_types():
    """fp32 queries over a cache in which other sequences, later tokens and freed slots hold NaN: the rows that see none are as the kernels'."""
    q, kc, vc, meta = _setup([0, 3, 64], [5000, 70, 90], 16, 8, 2, 128, 49)
    want, tol = _want(q, kc, vc, meta, 0.1)
    nan = torch.full((1, 2, 128), float("nan"), device=DEV, dtype=torch.bfloat16)
    for b, t in ((0, 3), (1, 69), (1, 71), (2, 80)):
        ops.write_kv_int4(nan, nan, kc, vc, (meta.block_table[b, t // 16].long() * 16 + t % 16).view(1))
    rows = [0, 1, *range(3, 3 + 54)]                              # token 69 is the second sequence's last, 80 the third's 55th new one
    f32, own = ops.paged_attention_int4(q.float(), kc, vc, meta, 0.1), ops.paged_attention_int4(q, kc, vc, meta, 0.1)
    for out in (f32, own):
        _check(out[rows], want[rows], tol[rows])
        rest = torch.ones(len(q), dtype=torch.bool)
        rest[rows] = False
        assert out[rest].isnan().all()


@pytest.mark.parametrize("method", ["eagle", "draft_model", "ngram"])
def test_engine_drafts_over_a_4_bit_cache(method):
    """Drafts keep their own pages beside the model's; blocks counted by what memory holds; repeated prompts come from the prefix cache (not with a
    draft model, whose catching up over whole prompts does not fit into a step)."""
    import numpy as np
    from vllm_ascend_b200.config import ModelConfig
    from vllm_ascend_b200.engine.llm import LLM
    from vllm_ascend_b200.engine.request import SamplingParams
    cfg = ModelConfig(name="t", architecture="Qwen3ForCausalLM", vocab_size=2048, hidden_size=512, intermediate_size=1024,
                      num_hidden_layers=3, num_attention_heads=8, num_key_value_heads=2, head_dim=128, qk_norm=True, rope_theta=1e6,
                      dtype="bfloat16", init_std=0.05)
    prompts = [np.tile(np.random.default_rng(i).integers(0, 2048, size=40), 8)[:n].tolist() for i, n in enumerate((300, 40, 133))]
    spec = {"method": method, "num_speculative_tokens": 3, **({"model": cfg} if method == "draft_model" else {})}
    llm = LLM(cfg, device="cuda", max_model_len=512, max_num_seqs=8, max_num_batched_tokens=256, kv_cache_dtype="int4",
              enable_prefix_caching=method != "draft_model", cudagraph_capture_sizes=[2, 4, 8], speculative_config=spec)
    runner = llm.engine.runner
    for _ in range(2):
        outs = llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=20, ignore_eos=True))
        assert all(len(o.outputs[0].token_ids) == 20 for o in outs)
    assert runner.spec_stats["draft_tokens"] > 0
    if method == "draft_model":                # the model itself drafts, over bf16 pages
        assert runner.spec_stats["accepted_tokens"] > 0 and runner.draft_bytes_per_block() * 9 == runner.kv_bytes_per_block() * 32
        assert all(t.dtype == torch.bfloat16 and t.shape[0] == runner.num_blocks for c in runner.proposer.kv_caches for t in c)
    assert all(t.dtype == torch.uint8 for c in runner.kv_caches for t in c)
    _native.check_status(torch.device(DEV))


@pytest.mark.parametrize("new,lens,Hq,Hkv", [([1], [45000], 8, 2), ([1, 1], [41001, 60000], 16, 8), ([300], [9000], 8, 2)])
def test_calls_at_once_whose_parts_join_through_memory(new, lens, Hq, Hkv, monkeypatch):
    """Every call has memory of its own for its parts' results: two streams, and a captured prompt replayed beside them.  Decodes that a graph
    holds join in clusters."""
    from vllm_ascend_b200.ops import kv_int4
    asked, results = [], kv_int4._results
    monkeypatch.setattr(kv_int4, "_results", lambda *a: asked.append(results(*a)) or asked[-1])
    sets = [_setup(new, lens, 128, Hq, Hkv, 128, seed) for seed in (50, 51)]
    want = [ops.paged_attention_int4(*s, 0.09) for s in sets]
    assert len(asked) == 2 and asked[0].data_ptr() != asked[1].data_ptr()
    for s, w in zip(sets, want):
        _check(w, *_want(*s, 0.09))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = ops.paged_attention_int4(*sets[0], 0.09)
    assert len(asked) == (2 if max(new) == 1 else 3)
    replayed.zero_()
    asked.clear()
    torch.cuda.synchronize()
    sides, got = [torch.cuda.Stream() for _ in range(3)], [[], []]
    for _ in range(20):
        for i, s in enumerate(sets):
            with torch.cuda.stream(sides[i]):
                got[i].append(ops.paged_attention_int4(*s, 0.09))
        with torch.cuda.stream(sides[2]):
            graph.replay()
    torch.cuda.synchronize()
    assert len(asked) == 40
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
    if max(new) > 1:
        assert torch.equal(replayed, want[0])
    else:
        _check(replayed, *_want(*sets[0], 0.09))
    _native.check_status(torch.device(DEV))
