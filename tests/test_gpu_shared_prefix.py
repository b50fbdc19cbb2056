"""Attention of batches that share prefixes, on the GPU."""
import pytest
import torch

from shared_prefix_cases import Batch

pytestmark = pytest.mark.gpu


def _ops():
    from vllm_ascend_b200 import ops
    return ops


GROUPS = {
    "one beam, one key": [(0, [(1, 1)])],
    "one prompt, four beams": [(1000, [(20, 1), (20, 1), (20, 1), (20, 1)])],
    "prefix alone": [(256, [(1, 1), (1, 1)])],
    "prefix inside a tile": [(77, [(3, 1), (130, 1)])],
    "odd prefixes": [(129, [(1, 1), (40, 1), (255, 1)]), (15, [(2, 1)]), (640, [(17, 1)] * 5)],
    "no prefix": [(0, [(300, 1), (1, 1)]), (0, [(129, 1)])],
    "drafts": [(200, [(5, 4), (9, 3), (4, 4)]), (31, [(2, 2), (150, 1)])],
    "many beams": [(700, [(33, 1)] * 40)],
    "more than two tiles of rows": [(500, [(9, 1)] * 90)],
    "prompts behind a prefix": [(300, [(150, 150), (70, 70), (260, 200)])],
    "unequal": [(2900, [(1, 1)]), (16, [(700, 1), (3, 1)])],
    "many groups": [(128, [(5, 1), (6, 1)])] * 60,
}
LAYOUTS = [(32, 8, 128, 128), (8, 1, 128, 16), (28, 4, 64, 16), (6, 2, 128, 32), (16, 16, 64, 64), (64, 8, 128, 128), (4, 4, 128, 8), (96, 1, 64, 256),
           (3, 1, 128, 128), (10, 2, 64, 128)]


@pytest.mark.parametrize("name", GROUPS)
@pytest.mark.parametrize("heads,kv_heads,dim,page", LAYOUTS[:3])
def test_batches(name, heads, kv_heads, dim, page):
    b = Batch(GROUPS[name], heads, kv_heads, dim, page, device="cuda")
    b.check(b.run(_ops()))


@pytest.mark.parametrize("heads,kv_heads,dim,page", LAYOUTS[3:])
@pytest.mark.parametrize("name", ["odd prefixes", "drafts", "more than two tiles of rows"])
def test_head_layouts(name, heads, kv_heads, dim, page):
    b = Batch(GROUPS[name], heads, kv_heads, dim, page, device="cuda", order="tokens", seed=3)
    b.check(b.run(_ops()))


def test_sequences_in_no_group_and_rows_behind_the_last():
    b = Batch(GROUPS["odd prefixes"], 8, 2, 128, 16, alone=[(40, 1), (129, 2)], device="cuda", pad_rows=5)
    b.check(b.run(_ops()))
    out = torch.full_like(b.q, 7.0).contiguous()
    got = b.run(_ops(), out)
    assert got is out and out[b.rows:].eq(7).all()
    b.check(out)


def test_sequences_without_new_tokens_or_keys():
    b = Batch([(64, [(3, 1), (0, 0), (10, 2)]), (32, [(0, 0)])], 8, 2, 128, 16, device="cuda")
    b.check(b.run(_ops()))
    b.meta.seq_lens[2] = b.meta.seq_lens_cpu[2] = 0     # two new tokens, no key
    b.lens[2] = 0
    b.keys[2], b.values[2] = b.keys[2][:0], b.values[2][:0]
    out = b.run(_ops())
    assert out[1:].eq(0).all() and out[0].isfinite().all()


def test_long_prefixes_join_many_pieces():
    b = Batch([(20000, [(130, 1), (5, 1), (700, 1)])], 8, 2, 128, 128, device="cuda", std=2.0)
    b.check(b.run(_ops()))


def test_large_scores():
    b = Batch(GROUPS["one prompt, four beams"], 8, 2, 128, 128, device="cuda", std=12.0)
    b.check(b.run(_ops()))
    b = Batch(GROUPS["drafts"], 28, 4, 64, 16, device="cuda", std=12.0)
    b.check(b.run(_ops()))


@pytest.mark.parametrize("dtype,dim,page", [(torch.float32, 128, 16), (torch.float16, 64, 16), (torch.bfloat16, 40, 16), (torch.bfloat16, 128, 12)])
def test_other_types_and_sizes(dtype, dim, page):
    b = Batch(GROUPS["odd prefixes"], 4, 2, dim, page, device="cuda", dtype=dtype)
    b.check(b.run(_ops()))


def test_views():
    b = Batch(GROUPS["odd prefixes"], 8, 2, 128, 16, device="cuda")
    want = b.run(_ops())
    wide = torch.full((b.table.shape[0], b.table.shape[1] + 3), 10 ** 6, dtype=torch.int32, device="cuda")
    wide[:, 2:-1] = b.meta.block_table
    b.meta.block_table = wide[:, 2:-1]
    lens = torch.zeros((len(b.lens), 2), dtype=torch.int32, device="cuda")
    lens[:, 1] = b.meta.seq_lens
    b.meta.seq_lens = lens[:, 1]
    out = torch.empty((b.rows, 8, 200), dtype=torch.bfloat16, device="cuda")[..., 30:158]
    assert torch.equal(b.run(_ops(), out), want)
    turned = b.k_cache.contiguous()                     # keys by tokens, values by heads
    got = _ops().paged_attention_shared(b.q, turned, b.v_cache, b.meta, b.plan(_ops()), b.scale)
    assert torch.equal(got, want)
    odd = torch.empty(b.q.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(b.q.shape)
    odd.copy_(b.q)
    assert torch.equal(_ops().paged_attention_shared(odd, b.k_cache, b.v_cache, b.meta, b.plan(_ops()), b.scale), want)


def test_results_repeat_and_two_streams_agree():
    ops = _ops()
    sets = [Batch(GROUPS[n], 32, 8, 128, 128, device="cuda", seed=i) for i, n in enumerate(("one prompt, four beams", "unequal"))]
    plans = [b.plan(ops) for b in sets]

    def call(b, plan):
        return ops.paged_attention_shared(b.q, b.k_cache, b.v_cache, b.meta, plan, b.scale)
    want = [call(b, p) for b, p in zip(sets, plans)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(10):
        got = []
        for b, p, s in zip(sets, plans, streams):
            with torch.cuda.stream(s):
                got.append(call(b, p))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_a_captured_plan_follows_its_lengths():
    ops = _ops()
    long = Batch([(900, [(200, 1), (100, 1), (7, 1), (300, 1)])], 32, 8, 128, 128, device="cuda")
    short = Batch([(256, [(40, 1), (1, 1)]), (128, [(5, 1), (90, 1)])], 32, 8, 128, 128, device="cuda", seed=5)
    starts = torch.zeros(3, dtype=torch.int32, device="cuda")
    prefixes = torch.zeros(2, dtype=torch.int32, device="cuda")
    k, v = (torch.zeros_like(t) for t in (long.k_cache, long.v_cache))
    q = long.q.clone()

    def load(b):
        n = b.starts.numel()
        starts.fill_(4)
        starts[:n] = b.starts
        prefixes.zero_()
        prefixes[:n - 1] = b.prefixes
        long.meta.seq_lens.copy_(b.meta.seq_lens)
        long.meta.block_table.fill_(10 ** 6)
        long.meta.block_table[:, :b.table.shape[1]] = b.meta.block_table
        k[:b.k_cache.shape[0]] = b.k_cache
        v[:b.v_cache.shape[0]] = b.v_cache
        q.copy_(b.q)
    lens = long.meta.seq_lens.clone()
    table = long.meta.block_table.clone()
    load(long)
    long.meta.block_table.copy_(table)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        plan = ops.plan_shared_prefix(long.meta, starts, prefixes, 32, 8)
        outs = [ops.paged_attention_shared(q, k, v, long.meta, plan, long.scale) for _ in range(2)]
    for b in (long, short, long):
        if b is short:
            load(short)
        else:
            load(long)
            long.meta.seq_lens.copy_(lens)
            long.meta.block_table.copy_(table)
        graph.replay()
        torch.cuda.synchronize()
        for o in outs:
            b.check(o)


def test_bad_pages_and_starts_are_reported():
    from vllm_ascend_b200 import _native
    for at in ((0, 0), (1, 9)):
        b = Batch(GROUPS["one prompt, four beams"], 8, 2, 128, 128, device="cuda")
        col = at[1] if at[0] == 0 else (1000 + 19) // 128
        b.meta.block_table[at[0], col] = -5
        b.run(_ops())
        torch.cuda.synchronize()
        with pytest.raises(_native.NativeError, match="BAD_INDEX"):
            _native.check_status(b.q.device)
    b = Batch(GROUPS["drafts"], 8, 2, 128, 16, device="cuda")
    for starts in ([0, 6, 5], [-1, 3, 5], [0, 3, 9]):
        b.starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        out = torch.full((b.rows, 8, 128), 3.0, dtype=torch.bfloat16, device="cuda")
        b.run(_ops(), out)
        torch.cuda.synchronize()
        with pytest.raises(_native.NativeError, match="BAD_INDEX"):
            _native.check_status(b.q.device)
        assert out.eq(3).all()


@pytest.mark.parametrize("prefix,seqs", [(128, 64), (100, 33), (16, 70)])
def test_short_prefixes_of_many_sequences(prefix, seqs):
    b = Batch([(prefix, [(1 + 37 * i % 150, 1) for i in range(seqs)])], 32, 8, 128, 16, device="cuda", seed=3)
    b.check(b.run(_ops()))


def test_lengths_that_no_cache_holds_are_reported():
    from vllm_ascend_b200 import _native
    b = Batch(GROUPS["one prompt, four beams"], 8, 8, 128, 128, device="cuda")
    b.meta.seq_lens.fill_(2 ** 31 - 200)
    b.prefixes = torch.zeros_like(b.prefixes)
    out = torch.full((b.rows, 8, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    b.run(_ops(), out)
    torch.cuda.synchronize()
    with pytest.raises(_native.NativeError, match="BAD_INDEX"):
        _native.check_status(b.q.device)
    assert out.eq(3).all()


def test_a_plan_outlives_its_owner_on_another_stream():
    ops = _ops()
    b = Batch(GROUPS["one prompt, four beams"], 32, 8, 128, 128, device="cuda")
    want = b.run(ops)
    side = torch.cuda.Stream()
    for _ in range(5):
        plan = b.plan(ops)
        size = plan.table.numel()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [ops.paged_attention_shared(b.q, b.k_cache, b.v_cache, b.meta, plan, b.scale) for _ in range(8)]
        del plan
        junk = [torch.full((size,), -1, dtype=torch.int32, device="cuda") for _ in range(4)]      # would take its place
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for x in got)
        del junk
