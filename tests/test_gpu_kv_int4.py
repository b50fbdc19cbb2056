"""4-bit cache on the GPU: stored bytes against the reference's, rows read back, attention of few rows and of prompts over it.

Attention is compared with fp64 attention over the values that the cache stands for.  Bound of an element, from the number types: the
kernels round probabilities to bf16 (half a step, 2^-8) before they weight values, and the result (2^-8); scores are fp32 sums of D
products (D 2^-24 of the largest sum of magnitudes, doubled for the products of the exponent's argument), which moves a probability by
as much, and the sum that it is divided by by as much again."""
import numpy as np
import pytest
import torch

from vllm_ascend_b200 import _native, batch_invariant, ops
from vllm_ascend_b200.attention.metadata import metadata_from_tensors
from vllm_ascend_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _caches(blocks, page, H, D, device=DEV):
    return tuple(ops.alloc_kv_cache_int4(blocks, page, H, D, device) for _ in "kv")


def _batch(new, lens, page, g):
    pages = [max(1, -(-n // page)) for n in lens]
    order = torch.randperm(sum(pages) + 2, generator=g).int()
    table = torch.full((len(new), max(pages)), -7, dtype=torch.int32)       # entries behind a sequence's pages are not read
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    return table.to(DEV), sum(pages) + 2


def _meta(new, lens, table, Hq, Hkv, D):
    cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device=DEV)
    return metadata_from_tensors(cu, torch.tensor(lens, dtype=torch.int32, device=DEV), table, max(new), max(lens), Hq, Hkv, D)


def _setup(new, lens, page, Hq, Hkv, D, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    table, blocks = _batch(new, lens, page, g)
    kc, vc = _caches(blocks, page, Hkv, D)
    k, v = (torch.randn(blocks * page, Hkv, D, generator=g).to(DEV, torch.bfloat16) for _ in "kv")
    k = k * spread
    ops.write_kv_int4(k, v, kc, vc, torch.arange(blocks * page, device=DEV))
    q = torch.randn(sum(new), Hq, D, generator=g).to(DEV, torch.bfloat16)
    return q, kc, vc, _meta(new, lens, table, Hq, Hkv, D)


def _want(q, kc, vc, meta, scale, window=0, causal=True):
    """fp64 results and the bound of every element."""
    T, Hq, D = q.shape
    Hkv = kc.shape[1]
    bs = ref.kv_int4_block_size(kc, D)
    out, tol = torch.zeros(T, Hq, D, dtype=torch.float64, device=DEV), torch.zeros(T, Hq, D, dtype=torch.float64, device=DEV)
    cu, lens = meta.query_start_loc_cpu, meta.seq_lens_cpu
    for b in range(len(lens)):
        n, a = int(lens[b]), int(cu[b + 1] - cu[b])
        if n == 0 or a == 0:
            continue
        pos = torch.arange(n, device=DEV)
        at = meta.block_table[b].long()[pos // bs] * bs + pos % bs
        k, v = (t.double() for t in ref.read_kv_int4(kc, vc, at, D))
        mine = torch.arange(n - a, n, device=DEV).unsqueeze(1)
        off = (pos > mine) & causal
        if window:
            off |= pos <= mine - window
        for h in range(Hq):
            x, kh, vh = q[cu[b]:cu[b + 1], h].double(), k[:, h // (Hq // Hkv)], v[:, h // (Hq // Hkv)]
            s = (x @ kh.T * scale).masked_fill(off, float("-inf"))
            p = torch.softmax(s, -1)
            p = torch.where(off.all(-1, keepdim=True), 0.0, p)
            o = p @ vh
            moved = 2 * (D + 4) * 2.0 ** -24 * float((x.abs() @ kh.nan_to_num(0.0).abs().T).max()) * scale
            out[cu[b]:cu[b + 1], h] = o
            tol[cu[b]:cu[b + 1], h] = (2.0 ** -8 + 2 * moved) * (p @ vh.abs()) * (1 + 2.0 ** -7) + 2.0 ** -8 * o.abs() + 1e-30
    return out, tol


def _check(got, want, tol):
    off = (got.double() - want).abs() - tol
    assert torch.isfinite(got).all() and float(off.max()) <= 0.0, float(((off + tol) / tol.clamp_min(1e-30)).max())


# ---------------------------------------------------------------- rows in and out
@pytest.mark.parametrize("D,page,H,T", [(128, 128, 8, 1), (128, 128, 8, 700), (64, 16, 1, 333), (64, 48, 3, 17), (128, 256, 5, 129), (128, 16, 40, 37),
                                        (64, 16, 33, 1000), (128, 128, 2, 9000)])
def test_bytes_of_stored_rows(D, page, H, T):
    g = torch.Generator().manual_seed(D + T)
    blocks = T // page + 3
    rows = torch.randn(T, (4 + 2 * H) * D, generator=g) * torch.exp(3 * torch.randn(T, 1, generator=g))
    rows[::7] = (torch.randint(-14, 15, rows[::7].shape, generator=g) / 2)             # ties
    rows[3::11, :D] = 0
    rows = rows.to(torch.bfloat16)
    k, v = rows[:, 4 * D:(4 + H) * D].view(T, H, D), rows[:, (4 + H) * D:].view(T, H, D)
    slots = torch.randperm(blocks * page, generator=g)[:T]
    slots[T // 2:T // 2 + T // 9] = -1
    want = _caches(blocks, page, H, D, "cpu")
    ops.write_kv_int4(k, v, *want, slots)
    rd = rows.to(DEV)
    kd, vd = rd[:, 4 * D:(4 + H) * D].view(T, H, D), rd[:, (4 + H) * D:].view(T, H, D)
    got = _caches(blocks, page, H, D)
    ops.write_kv_int4(kd, vd, *got, slots.to(DEV))
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    back = ops.read_kv_int4(*got, slots.to(DEV), D)
    for a, b in zip(back, ops.read_kv_int4(*want, slots, D)):
        assert torch.equal(a.cpu(), b)
    _native.check_status(torch.device(DEV))


def test_bytes_at_the_edges_of_the_type():
    """Every bf16 magnitude as a group's largest, next to halves, thirds and sevenths of it, and NaN and infinities."""
    bits = torch.arange(0, 0x8000, dtype=torch.int32)
    top = bits.to(torch.int16).view(torch.bfloat16).float()
    part = torch.tensor([1, -1, 1 / 2, 1 / 3, 1 / 7, -1 / 14, 3 / 14, 5 / 14, 0.999, -0.93, 0.786, 0.0714, 0, 0.5, -0.357, 0.0715] * 2)
    x = (top.unsqueeze(1) * part).to(torch.bfloat16)
    x[:, 0] = bits.to(torch.int16).view(torch.bfloat16)
    x = x.view(-1, 1, 64)
    T = x.shape[0]
    want, got = _caches(T // 128, 128, 1, 64, "cpu"), _caches(T // 128, 128, 1, 64)
    ops.write_kv_int4(x, -x, *want, torch.arange(T))
    ops.write_kv_int4(x.to(DEV), -x.to(DEV), *got, torch.arange(T, device=DEV))
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    slots = torch.arange(T)
    for a, b in zip(ops.read_kv_int4(*got, slots.to(DEV), 64), ops.read_kv_int4(*want, slots, 64)):
        assert torch.equal(a.cpu().isnan(), b.isnan()) and torch.equal(a.cpu().nan_to_num(0), b.nan_to_num(0))


def test_rows_of_odd_strides_int32_slots_and_other_types():
    g = torch.Generator().manual_seed(5)
    T, H, D = 9, 2, 64
    base = torch.randn(T, H, D + 3, generator=g).to(DEV, torch.bfloat16)
    k, v = base[:, :, 3:], base.flip(2)[:, :, :D].transpose(0, 1).contiguous().transpose(0, 1)
    for dtype in (torch.bfloat16, torch.float32):
        want, got = _caches(1, 16, H, D, "cpu"), _caches(1, 16, H, D)
        slots = torch.arange(T, dtype=torch.int32) + 3
        ops.write_kv_int4(k.to(dtype), v.to(dtype), *got, slots.to(DEV))
        ops.write_kv_int4(k.to(dtype).cpu(), v.to(dtype).cpu(), *want, slots)
        for a, b in zip(got, want):
            assert torch.equal(a.cpu(), b)


def test_slots_outside_of_the_cache_are_reported():
    kc, vc = _caches(2, 16, 1, 64)
    x = torch.ones(2, 1, 64, device=DEV, dtype=torch.bfloat16)
    ops.write_kv_int4(x, x, kc, vc, torch.tensor([32, 5], device=DEV))
    with pytest.raises(_native.NativeError, match="BAD_INDEX"):
        _native.check_status(torch.device(DEV))
    k, _ = ops.read_kv_int4(kc, vc, torch.tensor([5, 1 << 40], device=DEV), 64)
    with pytest.raises(_native.NativeError, match="BAD_INDEX"):
        _native.check_status(torch.device(DEV))
    assert k[0].eq(7 * 19 / 128).all()                # 19 / 128 is the first number of five bits from 1 / 7 on
    assert not k[1].any() and not kc[1].any()


# ---------------------------------------------------------------- attention of few rows
@pytest.mark.parametrize("Hq,Hkv,D,page", [(32, 8, 128, 128), (8, 1, 128, 16), (4, 4, 128, 64), (28, 4, 64, 16), (16, 1, 128, 48), (6, 2, 64, 128),
                                           (24, 1, 64, 32), (40, 1, 128, 128)])
def test_decode(Hq, Hkv, D, page):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 400, 1337, 3001]
    q, kc, vc, meta = _setup([1] * len(lens), lens, page, Hq, Hkv, D, Hq + page)
    scale = D ** -0.5
    out = ops.paged_attention_int4(q, kc, vc, meta, scale)
    _check(out, *_want(q, kc, vc, meta, scale))
    _native.check_status(torch.device(DEV))


@pytest.mark.parametrize("each,Hq,Hkv,D,window,causal", [(2, 32, 8, 128, 0, True), (4, 32, 4, 128, 0, True), (5, 6, 2, 64, 0, True),
                                                         (3, 28, 4, 64, 40, True), (4, 8, 2, 128, 0, False), (1, 32, 8, 128, 100, True),
                                                         (2, 8, 8, 128, 1, True)])
def test_several_tokens_windows_and_open_masks(each, Hq, Hkv, D, window, causal):
    lens = [each, each + 1, 31, 32, 33, 100, 129, 777, 2050]
    q, kc, vc, meta = _setup([each] * len(lens), lens, 16, Hq, Hkv, D, each)
    out = ops.paged_attention_int4(q, kc, vc, meta, 0.11, causal=causal, window=window)
    _check(out, *_want(q, kc, vc, meta, 0.11, window, causal))


def test_one_long_sequence():
    q, kc, vc, meta = _setup([1], [70003], 128, 8, 2, 128, 3)
    out = ops.paged_attention_int4(q, kc, vc, meta, 128 ** -0.5)
    _check(out, *_want(q, kc, vc, meta, 128 ** -0.5))


@pytest.mark.parametrize("lens,Hq,Hkv,D,each", [([9000], 8, 2, 128, 1), ([8001], 4, 1, 64, 1), ([12345, 3], 16, 8, 128, 1), ([9000, 0, 8100], 16, 8, 64, 1),
                                                ([9001], 16, 2, 128, 2)])
def test_wide_clusters(lens, Hq, Hkv, D, each):
    """Few long sequences: 14 or 16 parts, some without keys, joined by eight at a time."""
    q, kc, vc, meta = _setup([each] * len(lens), lens, 128, Hq, Hkv, D, 30)
    _check(ops.paged_attention_int4(q, kc, vc, meta, 0.1), *_want(q, kc, vc, meta, 0.1))
    _native.check_status(torch.device(DEV))


def test_growing_and_peaked_scores():
    """Keys whose scores climb along the sequence (every tile moves the maximum), and a score that outweighs all others."""
    D, n = 128, 1500
    q, kc, vc, meta = _setup([1, 1], [n, n], 64, 8, 2, D, 4)
    k = torch.ones(n, 2, D, device=DEV, dtype=torch.bfloat16) * torch.linspace(0.1, 12, n, device=DEV).view(n, 1, 1).bfloat16()
    v = torch.randn(n, 2, D, device=DEV, dtype=torch.bfloat16)
    pos = torch.arange(n, device=DEV)
    for b in range(2):
        ops.write_kv_int4(k if b == 0 else k.flip(0).contiguous(), v, kc, vc, meta.block_table[b].long()[pos // 64] * 64 + pos % 64)
    q = q.abs()
    out = ops.paged_attention_int4(q, kc, vc, meta, 0.5)
    _check(out, *_want(q, kc, vc, meta, 0.5))


def test_tokens_that_see_no_key_and_rows_behind_the_last_sequence():
    q, kc, vc, meta = _setup([1, 3, 1], [0, 1, 40], 16, 8, 2, 128, 6)
    q = torch.cat([q, torch.full((3, 8, 128), float("nan"), device=DEV, dtype=torch.bfloat16)])
    out = torch.full_like(q, 7.0)
    got = ops.paged_attention_int4(q, kc, vc, meta, 0.1, out=out)
    assert got is out and out[5:].eq(7).all()
    assert not out[0].any() and not out[1:3].any()                # an empty sequence; new tokens in front of the first key
    want, tol = _want(q[:5], kc, vc, meta, 0.1)
    _check(out[:5], want, tol)


def test_what_lies_outside_of_a_sequence_does_not_matter():
    """NaN rows in the slots behind the last token, in front of a window and in later tokens of the same step."""
    D, page, each = 128, 32, 3
    lens = [37, 70, 129]
    q, kc, vc, meta = _setup([each] * 3, lens, page, 8, 2, D, 8)
    for window in (0, 20):
        want, tol = _want(q, kc, vc, meta, 0.1, window)
        bad_k, bad_v = kc.clone(), vc.clone()
        nan = torch.full((1, 2, D), float("nan"), device=DEV, dtype=torch.bfloat16)
        spots = []
        for b, n in enumerate(lens):
            last = -(-n // page) * page
            spots += [(b, t) for t in range(n, last)] + [(b, t) for t in range(0, n - each - window + 1) if window]
        for b, t in spots:
            slot = meta.block_table[b, t // page].long().view(1) * page + t % page
            ops.write_kv_int4(nan, nan, bad_k, bad_v, slot)
        out = ops.paged_attention_int4(q, bad_k, bad_v, meta, 0.1, window=window)
        _check(out, want, tol)
        # a NaN in the step's last token: the tokens in front of it stay as they are, its own row is NaN where the group is
        slots = torch.stack([meta.block_table[b, (n - 1) // page].long() * page + (n - 1) % page for b, n in enumerate(lens)])
        rows = torch.ones((3, 2, D), device=DEV, dtype=torch.bfloat16)
        rows[:, 0, 40] = float("inf")
        ops.write_kv_int4(rows, rows, bad_k, bad_v, slots)
        ones = torch.ones_like(rows)
        ops.write_kv_int4(ones, ones, kc, vc, slots)
        want, tol = _want(q, kc, vc, meta, 0.1, window)
        ops.write_kv_int4(ones, rows, kc, vc, slots)
        out = ops.paged_attention_int4(q, kc, vc, meta, 0.1, window=window)
        for b in range(3):
            a = each * b
            _check(out[a:a + 2], want[a:a + 2], tol[a:a + 2])
            assert out[a + 2, :4, 32:64].isnan().all()
            keep = [c for c in range(D) if not 32 <= c < 64]
            _check(out[a + 2, :4, keep], want[a + 2, :4, keep], tol[a + 2, :4, keep])
            _check(out[a + 2, 4:], want[a + 2, 4:], tol[a + 2, 4:])
        out = ops.paged_attention_int4(q, bad_k, bad_v, meta, 0.1, window=window)
        assert torch.isfinite(out[[0, 1, 3, 4, 6, 7]]).all() and out[[2, 5, 8], :4].isnan().all()
        q, kc, vc, meta = _setup([each] * 3, lens, page, 8, 2, D, 9)


def test_pages_outside_of_the_cache_are_reported():
    q, kc, vc, meta = _setup([1, 1], [300, 40], 16, 8, 2, 128, 11)
    good = ops.paged_attention_int4(q, kc, vc, meta, 0.1)
    meta.block_table[0, 7] = kc.shape[0]
    out = ops.paged_attention_int4(q, kc, vc, meta, 0.1)
    with pytest.raises(_native.NativeError, match="BAD_INDEX"):
        _native.check_status(torch.device(DEV))
    assert torch.equal(out[1], good[1])


def test_given_outputs_strides_and_other_types():
    q, kc, vc, meta = _setup([1, 2], [50, 90], 16, 8, 2, 64, 12)
    want, tol = _want(q, kc, vc, meta, 0.2)
    rows = torch.zeros(3, 8 * 64 + 24, device=DEV, dtype=torch.bfloat16)
    rows[:, 8:8 + 512] = q.view(3, 512)
    strided = rows[:, 8:8 + 512].view(3, 8, 64)
    out = torch.zeros(3, 8, 130, device=DEV, dtype=torch.bfloat16)[:, :, 1:65]
    assert ops.paged_attention_int4(strided, kc, vc, meta, 0.2, out=out) is out
    _check(out, want, tol)
    odd = torch.zeros(3, 8, 65, device=DEV, dtype=torch.bfloat16)[:, :, 1:].copy_(q)
    _check(ops.paged_attention_int4(odd, kc, vc, meta, 0.2), want, tol)
    f32 = ops.paged_attention_int4(q.float(), kc, vc, meta, 0.2)
    assert f32.dtype == torch.float32 and float((f32.double() - want).abs().max()) < 1e-4


@pytest.fixture(params=["prompts", "few rows"])
def kernel(request, monkeypatch):
    """Sequences that could go to either kernel go to this one."""
    from vllm_ascend_b200.ops import kv_int4
    monkeypatch.setattr(kv_int4, "_prompt_us", lambda *a: 1e9 if request.param == "few rows" else -1e9)
    kv_int4._plan.cache_clear()
    yield request.param
    kv_int4._plan.cache_clear()


def test_modes_with_a_fixed_order_of_sums(monkeypatch):
    """A sequence's row has the same bits alone and in a batch."""
    lens = [1000, 64, 513]
    q, kc, vc, meta = _setup([1] * 3, lens, 32, 8, 2, 128, 13)
    monkeypatch.setattr("vllm_ascend_b200.ops.kv_int4.fixed_sums", lambda: True)
    out = ops.paged_attention_int4(q, kc, vc, meta, 0.1)
    for b in range(3):
        one = _meta([1], [lens[b]], meta.block_table[b:b + 1], 8, 2, 128)
        assert torch.equal(ops.paged_attention_int4(q[b:b + 1], kc, vc, one, 0.1), out[b:b + 1])


def test_modes_with_a_fixed_order_of_sums_over_mixed_batches(monkeypatch):
    """Neither do short sequences behind long ones change with their neighbours."""
    new, lens = [1, 200, 3, 1, 90], [700, 200, 503, 64, 1000]
    q, kc, vc, meta = _setup(new, lens, 32, 8, 2, 128, 15)
    monkeypatch.setattr("vllm_ascend_b200.ops.kv_int4.fixed_sums", lambda: True)
    out = ops.paged_attention_int4(q, kc, vc, meta, 0.1)
    _check(out, *_want(q, kc, vc, meta, 0.1))
    cu = meta.query_start_loc_cpu
    for b in range(5):
        one = _meta(new[b:b + 1], lens[b:b + 1], meta.block_table[b:b + 1], 8, 2, 128)
        assert torch.equal(ops.paged_attention_int4(q[cu[b]:cu[b + 1]], kc, vc, one, 0.1), out[cu[b]:cu[b + 1]])


def test_sequences_without_new_tokens_in_front(kernel):
    q, kc, vc, meta = _setup([0, 0, 200, 0], [60000, 5, 300, 9], 128, 8, 2, 128, 34)
    _check(ops.paged_attention_int4(q, kc, vc, meta, 0.1), *_want(q, kc, vc, meta, 0.1))


@pytest.mark.parametrize("most", [None, 1 << 20])
@pytest.mark.parametrize("new,lens", [([1, 90, 3], [41000, 9000, 8]), ([300], [9000])])
def test_memory_of_parts(new, lens, most, kernel, monkeypatch):
    """Only of the rows that have parts, and no more than there may be."""
    from vllm_ascend_b200.ops import kv_int4
    if most:
        monkeypatch.setattr(kv_int4, "MOST_BYTES", most)
    asked, empty = [], torch.empty
    q, kc, vc, meta = _setup(new, lens, 128, 8, 2, 128, 33)
    monkeypatch.setattr(kv_int4.torch, "empty", lambda *a, **kw: asked.append(a[0]) or empty(*a, **kw))
    out = ops.paged_attention_int4(q, kc, vc, meta, 0.1)
    monkeypatch.undo()
    assert all(4 * n <= (most or 256 << 20) for n in asked) and (most or asked or kernel == "few rows")
    _check(out, *_want(q, kc, vc, meta, 0.1))


@pytest.mark.parametrize("new,lens", [([1], [40000]), ([300], [9000])])
def test_calls_on_two_streams_at_once(new, lens, kernel):
    """Sequences in parts that join through memory: every call, and every graph, has its own."""
    sets = [_setup(new, lens, 128, 8, 2, 128, seed) for seed in (16, 17)]
    want = [ops.paged_attention_int4(*s, 0.09) for s in sets]
    torch.cuda.synchronize()
    sides, graphs, got, replayed = [torch.cuda.Stream() for _ in sets], [], [[], []], []
    for _ in range(20):
        for i, s in enumerate(sets):
            with torch.cuda.stream(sides[i]):
                got[i].append(ops.paged_attention_int4(*s, 0.09))
    torch.cuda.synchronize()
    for i, s in enumerate(sets):
        assert all(torch.equal(x, want[i]) for x in got[i])
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            replayed.append(ops.paged_attention_int4(*s, 0.09))
    for x in replayed:
        x.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for i, graph in enumerate(graphs):
            with torch.cuda.stream(sides[i]):
                graph.replay()
    torch.cuda.synchronize()
    # a captured call may split a sequence otherwise (by what its table holds)
    for x, s in zip(replayed, sets):
        _check(x, *_want(*s, 0.09))


@pytest.mark.parametrize("D,window", [(64, 0), (128, 0), (64, 5000)])
def test_many_sequences_of_all_lengths(D, window):
    """In parts where the host knows the lengths, whole in a graph that is replayed with others."""
    lens = [6500, 1, 100, 2047, 2048, 4095, 4096, 4097, 6145, 6500, 0] * 3
    q, kc, vc, meta = _setup([1] * 33, lens, 128, 8, 8, D, 19)
    out = ops.paged_attention_int4(q, kc, vc, meta, 0.1, window=window)
    _check(out, *_want(q, kc, vc, meta, 0.1, window))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_attention_int4(q, kc, vc, meta, 0.1, window=window)
    other = torch.tensor([max(0, n - 3 * i) for i, n in enumerate(lens)], dtype=torch.int32)
    meta.seq_lens.copy_(other)
    meta.seq_lens_cpu = other.numpy()
    graph.replay()
    torch.cuda.synchronize()
    _check(out, *_want(q, kc, vc, meta, 0.1, window))
    _native.check_status(torch.device(DEV))


@pytest.mark.parametrize("new", [[1, 1], [100, 60]])
def test_row_numbers_beyond_the_rows_are_reported(new, kernel):
    q, kc, vc, meta = _setup(new, [200, 300], 32, 8, 2, 128, 18)
    want, tol = _want(q, kc, vc, meta, 0.1)
    meta.query_start_loc[2] += 1
    out = torch.full_like(q, 5.0)
    ops.paged_attention_int4(q, kc, vc, meta, 0.1, out=out)
    _check(out[:new[0]], want[:new[0]], tol[:new[0]])
    assert out[new[0]:].eq(5).all()
    with pytest.raises(_native.NativeError, match="BAD_INDEX"):
        _native.check_status(torch.device(DEV))


def test_graph_replay_with_other_lengths_and_another_stream():
    lens = [700, 1, 2000]
    q, kc, vc, meta = _setup([1] * 3, lens, 128, 32, 8, 128, 14)
    ops.paged_attention_int4(q, kc, vc, meta, 0.09)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_attention_int4(q, kc, vc, meta, 0.09)
    other = torch.tensor([333, 90, 1999], dtype=torch.int32)
    meta.seq_lens.copy_(other)
    meta.seq_lens_cpu = other.numpy()
    graph.replay()
    torch.cuda.synchronize()
    want, tol = _want(q, kc, vc, meta, 0.09)
    _check(out, want, tol)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.paged_attention_int4(q, kc, vc, meta, 0.09)
    side.synchronize()
    assert torch.equal(again, out)


# ---------------------------------------------------------------- prompts
@pytest.mark.parametrize("Hq,Hkv,D,page,window,causal", [
    (8, 2, 128, 128, 0, True), (4, 4, 128, 16, 0, True), (28, 4, 64, 16, 0, True), (16, 1, 128, 48, 0, True), (6, 2, 64, 128, 0, True),
    (8, 1, 128, 64, 100, True), (8, 2, 64, 32, 1, True), (4, 2, 128, 256, 0, False), (5, 1, 128, 32, 300, True), (2, 2, 64, 128, 77, True)])
def test_prompts(Hq, Hkv, D, page, window, causal, kernel):
    tile = 128 // (Hq // Hkv)
    new = [20, tile - 1, tile, tile + 1, 2 * tile, 2 * tile + 1, 300, 17, 3]
    old = [0, 5, 0, 200, 129, 0, 77, 640, 250]
    q, kc, vc, meta = _setup(new, [a + b for a, b in zip(new, old)], page, Hq, Hkv, D, Hq + page + window)
    scale = 1.3 * D ** -0.5
    out = ops.paged_attention_int4(q, kc, vc, meta, scale, causal=causal, window=window)
    _check(out, *_want(q, kc, vc, meta, scale, window, causal))
    _native.check_status(torch.device(DEV))


@pytest.mark.parametrize("D,Hq,Hkv", [(128, 8, 2), (64, 16, 4)])
def test_mixed_batches(D, Hq, Hkv, kernel):
    """Decodes in front of prompts, a short sequence behind them, tokens behind the last sequence."""
    new, old = [1, 1, 1, 2, 130, 1, 700, 9], [5, 300, 1000, 64, 0, 90, 333, 2000]
    q, kc, vc, meta = _setup(new, [a + b for a, b in zip(new, old)], 32, Hq, Hkv, D, 21)
    want, tol = _want(q, kc, vc, meta, 0.1)
    q = torch.cat([q, torch.full((5, Hq, D), float("nan"), device=DEV, dtype=torch.bfloat16)])
    out = torch.full_like(q, 3.0)
    ops.paged_attention_int4(q, kc, vc, meta, 0.1, out=out)
    _check(out[:-5], want, tol)
    assert out[-5:].eq(3).all()


def test_a_long_portion_behind_a_long_context(kernel):
    q, kc, vc, meta = _setup([333], [20333], 128, 8, 2, 128, 22)
    _check(ops.paged_attention_int4(q, kc, vc, meta, 0.09), *_want(q, kc, vc, meta, 0.09))


def test_prompt_tokens_that_see_no_key(kernel):
    """More new tokens than keys: those in front of the first key get zeros."""
    q, kc, vc, meta = _setup([300, 40, 64], [20, 0, 64], 16, 8, 2, 128, 23)
    out = ops.paged_attention_int4(q, kc, vc, meta, 0.1)
    assert not out[:280].any() and not out[300:340].any()
    _check(out, *_want(q, kc, vc, meta, 0.1))


@pytest.mark.parametrize("window,D", [(0, 128), (200, 128), (0, 64)])
def test_nan_values_reach_the_prompt_rows_that_see_them(window, D, kernel):
    new, old, page = [260, 70], [500, 3], 32
    q, kc, vc, meta = _setup(new, [a + b for a, b in zip(new, old)], page, 8, 2, D, 24)
    spots = [(0, 10), (0, 300), (0, 500), (0, 640), (0, 758), (1, 2), (1, 60)]
    slots = torch.stack([meta.block_table[b, t // page].long() * page + t % page for b, t in spots])
    ones = torch.ones(len(spots), 2, D, device=DEV, dtype=torch.bfloat16)
    ops.write_kv_int4(ones, ones, kc, vc, slots)
    want, tol = _want(q, kc, vc, meta, 0.1, window)
    bad = ones.clone()
    bad[:, 1, 37] = float("nan")
    ops.write_kv_int4(ones, bad, kc, vc, slots)
    out = ops.paged_attention_int4(q, kc, vc, meta, 0.1, window=window)
    hit = torch.zeros_like(want, dtype=torch.bool)
    starts = [0, 260]
    for b, t in spots:
        pos = torch.arange(old[b], old[b] + new[b], device=DEV)
        sees = (pos >= t) & ((pos < t + window) if window else True)
        hit[starts[b]:starts[b] + new[b], 4:, 32:64] |= sees.view(-1, 1, 1)
    assert out.isnan().equal(hit)
    _check(torch.where(hit, 0.0, out), torch.where(hit, 0.0, want), tol)


def test_prompt_pages_outside_of_the_cache_are_reported(kernel):
    q, kc, vc, meta = _setup([200, 100], [300, 100], 16, 8, 2, 128, 25)
    good = ops.paged_attention_int4(q, kc, vc, meta, 0.1)
    meta.block_table[0, 7] = -3
    out = ops.paged_attention_int4(q, kc, vc, meta, 0.1)
    with pytest.raises(_native.NativeError, match="BAD_INDEX"):
        _native.check_status(torch.device(DEV))
    assert torch.equal(out[200:], good[200:])


# ---------------------------------------------------------------- as the engine uses it
def test_norm_rotation_and_store():
    """The model's call: rows are normed and rotated as for a bf16 cache, what the slots stand for is the quantised result."""
    T, Hq, Hkv, D = 37, 8, 2, 128
    g = torch.Generator().manual_seed(31)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).to(DEV, torch.bfloat16)
    wq, wk = (torch.rand(D, generator=g).to(DEV, torch.bfloat16) + 0.5 for _ in "qk")
    pos, slots = torch.arange(T, device=DEV) + 11, torch.randperm(128, generator=g)[:T].to(DEV)
    slots[5] = -1
    ang = torch.outer(torch.arange(64.0), 10000.0 ** (-torch.arange(0, D, 2) / D))
    cos_sin = torch.cat([ang.cos(), ang.sin()], -1).to(DEV)
    args = (pos, cos_sin, D, wq, wk, 1e-6)
    dense, rows = qkv.clone(), qkv.clone()
    kc, vc = (ops.alloc_kv_cache(4, 32, Hkv, D, torch.bfloat16, DEV) for _ in "kv")
    ops.qknorm_rope_kvwrite(dense, *args, kc, vc, slots, Hq, Hkv, D)
    k4, v4 = _caches(4, 32, Hkv, D)
    ops.qknorm_rope_kvwrite(rows, *args, k4, v4, slots, Hq, Hkv, D)
    assert torch.equal(rows, dense)
    want = _caches(4, 32, Hkv, D)
    k, v = (dense[:, a * D:(a + Hkv) * D].view(T, Hkv, D) for a in (Hq, Hq + Hkv))
    ops.write_kv_int4(k, v, *want, slots)
    assert torch.equal(k4, want[0]) and torch.equal(v4, want[1]) and k4.any()


@pytest.mark.parametrize("eager", [True, False])
def test_engine_over_a_4_bit_cache(eager):
    from vllm_ascend_b200.config import ModelConfig
    from vllm_ascend_b200.engine.llm import LLM
    from vllm_ascend_b200.engine.request import SamplingParams
    cfg = ModelConfig(name="t", architecture="Qwen3ForCausalLM", vocab_size=2048, hidden_size=512, intermediate_size=1024,
                      num_hidden_layers=3, num_attention_heads=8, num_key_value_heads=2, head_dim=128, qk_norm=True, rope_theta=1e6,
                      dtype="bfloat16", init_std=0.05)
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, 2048, size=n).tolist() for n in (150, 40, 333, 129)]
    llm = LLM(cfg, device="cuda", max_model_len=512, max_num_seqs=8, max_num_batched_tokens=256, num_gpu_blocks_override=40,
              enforce_eager=eager, cudagraph_capture_sizes=[2, 4, 8], kv_cache_dtype="int4")
    outs = llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=12, ignore_eos=True))
    assert all(len(o.outputs[0].token_ids) == 12 for o in outs)
    again = llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=12, ignore_eos=True))
    assert [o.outputs[0].token_ids for o in again] == [o.outputs[0].token_ids for o in outs]
    runner = llm.engine.runner
    assert eager or runner.stats["graph_replays"] > 0
    assert all(t.dtype == torch.uint8 and t.any() for pair in runner.kv_caches for t in pair)
    _native.check_status(torch.device(DEV))
