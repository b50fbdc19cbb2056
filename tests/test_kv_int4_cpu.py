"""4-bit cache on the host: the quantiser against its definition in whole numbers, the page layout byte by byte, what the operators
refuse, attention over the cache."""
import dataclasses
from fractions import Fraction

import numpy as np
import pytest
import torch

from vllm_ascend_b200 import ops
from vllm_ascend_b200.attention.metadata import metadata_from_tensors
from vllm_ascend_b200.ops import reference as ref


def _definition(group):
    """Scale and whole numbers of 32 finite numbers, in exact arithmetic."""
    x = [Fraction(float(v)) for v in group]
    top = max(abs(v) for v in x)
    if top == 0:
        return Fraction(0), [0] * len(x)
    e = -140
    while Fraction(31) * Fraction(2) ** e * 7 < top:              # scales of five bits: m 2^e, 16 <= m <= 31
        e += 1
    s = next(m * Fraction(2) ** e for m in range(1, 32) if 7 * m * Fraction(2) ** e >= top)
    s = min(max(s, Fraction(2) ** -80), Fraction(2) ** 34)
    return s, [min(max(round(v / s), -7), 7) for v in x]          # round(): ties to even


def _meta(new, lens, table, Hq, Hkv, D):
    cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
    return metadata_from_tensors(cu, torch.tensor(lens, dtype=torch.int32), table, max(new), max(lens), Hq, Hkv, D)


def test_quantiser_is_its_definition():
    g = torch.Generator().manual_seed(0)
    rows = [torch.randn(32, generator=g) * 10.0 ** s for s in (-20, -3, 0, 0, 0, 2, 20)]
    rows += [torch.arange(-16, 16).float() * 0.4375, torch.full((32,), 7.0), torch.zeros(32), torch.randint(-28, 29, (32,), generator=g) / 4]
    x = torch.stack(rows).to(torch.bfloat16)
    n, s = ref.kv_int4_quantise(x)
    for i in range(len(x)):
        want_s, want_n = _definition(x[i])
        assert Fraction(float(s[i, 0])) == want_s and n[i].tolist() == want_n, i
    assert (n.float() * s.float().repeat_interleave(32, -1)).to(torch.bfloat16).float().equal(n.float() * s.float().repeat_interleave(32, -1))


def test_quantiser_at_the_edges_of_the_type():
    x = torch.zeros(6, 64, dtype=torch.bfloat16)
    x[0, 3] = float("nan")
    x[1, 40] = float("-inf")
    x[2, :] = torch.finfo(torch.bfloat16).max
    x[3, 0] = 1e-40                                # subnormal
    x[4, 1] = -1.0
    n, s = ref.kv_int4_quantise(x)
    assert s[0, 0].isnan() and not n[0].any() and s[0, 1] == 0
    assert s[1, 1].isnan() and s[1, 0] == 0
    assert (s[2] == 2.0 ** 34).all() and (n[2] == 7).all()
    assert s[3, 0].float() == 2.0 ** -80                                  # the smallest scale: n is 0, within half a scale still
    assert (x[3, 0].double() - n[3, 0] * s[3, 0].double()).abs() <= s[3, 0].double() / 2
    assert s[5].eq(0).all() and not n[5].any() and n[4, 1] == -7


@pytest.mark.parametrize("D,page,H", [(64, 16, 1), (128, 48, 3), (128, 128, 2)])
def test_page_layout(D, page, H):
    g = torch.Generator().manual_seed(D + page)
    T = page + 5
    k, v = (torch.randn(T, H, D, generator=g).to(torch.bfloat16) for _ in "kv")
    kc, vc = (ops.alloc_kv_cache_int4(3, page, H, D, "cpu") for _ in "kv")
    assert kc.shape == (3, H, page * D * 9 // 16)
    slots = torch.randperm(3 * page, generator=g)[:T]
    slots[2] = -1
    ops.write_kv_int4(k, v, kc, vc, slots)
    for x, cache, values in ((k, kc, False), (v, vc, True)):
        n, s = ref.kv_int4_quantise(x)
        for t in (0, 1, 3, 4, T - 2, T - 1):
            blk, off = divmod(int(slots[t]), page)
            unit, i = divmod(off, 16)
            for h in (0, H - 1):
                mem = cache[blk, h, unit * 9 * D:(unit + 1) * 9 * D].tolist()
                scales = cache[blk, h, unit * 9 * D + 8 * D:(unit + 1) * 9 * D].view(torch.bfloat16)
                for ch in range(0, D, 2):
                    byte = int(n[t, h, ch]) + 8 + 16 * (int(n[t, h, ch + 1]) + 8)
                    if values:
                        chunk = ch // 16 ^ (2 * (i // 2 % 4) if D == 128 else i // 2 & 2)
                        assert mem[i // 2 * D + chunk * 16 + ch % 16 // 4 * 4 + i % 2 * 2 + ch % 4 // 2] == byte
                    else:
                        assert mem[i * D // 2 + ch // 2] == byte
                    assert scales[ch // 32 * 16 + i] == s[t, h, ch // 32]
    got = ops.read_kv_int4(kc, vc, slots, D)
    for x, y in zip((k, v), got):
        n, s = ref.kv_int4_quantise(x)
        want = (n.float() * s.float().repeat_interleave(32, -1)).to(torch.bfloat16)
        want[2] = 0
        assert y.equal(want)


@pytest.mark.parametrize("window,causal", [(0, True), (5, True), (0, False)])
def test_attention_over_the_cache(window, causal):
    g = torch.Generator().manual_seed(window)
    Hq, Hkv, D, page = 6, 2, 64, 16
    new, lens = [1, 4, 9], [33, 4, 20]
    table = torch.tensor([[5, 1, 2], [0, 7, 7], [3, 4, 7]], dtype=torch.int32)
    kc, vc = (ops.alloc_kv_cache_int4(8, page, Hkv, D, "cpu") for _ in "kv")
    k, v = (torch.randn(8 * page, Hkv, D, generator=g) for _ in "kv")
    ops.write_kv_int4(k, v, kc, vc, torch.arange(8 * page))
    q = torch.randn(sum(new), Hq, D, generator=g)
    out = ops.paged_attention_int4(q, kc, vc, _meta(new, lens, table, Hq, Hkv, D), D ** -0.5, causal=causal, window=window)
    kd, vd = (t.double() for t in ops.read_kv_int4(kc, vc, torch.arange(8 * page), D))
    row = 0
    for b, (a, n) in enumerate(zip(new, lens)):
        pos = torch.arange(n)
        at = table[b].long()[pos // page] * page + pos % page
        mine = torch.arange(n - a, n).unsqueeze(1)
        off = (pos > mine) & causal
        if window:
            off |= pos <= mine - window
        for h in range(Hq):
            s = (q[row:row + a, h].double() @ kd[at, h // 3].T * D ** -0.5).masked_fill(off, float("-inf"))
            want = torch.softmax(s, -1) @ vd[at, h // 3]
            assert (out[row:row + a, h].double() - want).abs().max() < 1e-5
        row += a


def test_refusals():
    k = torch.zeros(2, 2, 64)
    kc, vc = (ops.alloc_kv_cache_int4(2, 16, 2, 64, "cpu") for _ in "kv")
    slots = torch.zeros(2, dtype=torch.int64)
    for bad in (dict(dim=96), dict(dim=256), dict(block_size=24), dict(block_size=0)):
        with pytest.raises(ValueError, match="4-bit cache takes"):
            ops.alloc_kv_cache_int4(**{**dict(num_blocks=1, block_size=16, heads=1, dim=64, device="cpu"), **bad})
    write = ops.write_kv_int4
    for args, why in (((k, k[:1], kc, vc, slots), "not rows"), ((k, k.double(), kc, vc, slots), "not rows"),
                      ((k.long(), k.long(), kc, vc, slots), "not rows"), ((k[:, :1], k[:, :1], kc, vc, slots), "heads"),
                      ((k, k, kc, vc[:1], slots), "different sizes"), ((k, k, kc.view(torch.int8), vc, slots), "dense 4-bit"),
                      ((k, k, kc[:, :, :-1], vc, slots), "dense 4-bit"), ((k, k, kc, vc, slots[:1]), "slots"),
                      ((k, k, kc, vc, slots.float()), "slots"), ((k[..., :48], k[..., :48], kc, vc, slots), "takes heads")):
        with pytest.raises(ValueError, match=why):
            write(*args)
    with pytest.raises(ValueError, match="slots"):
        ops.read_kv_int4(kc, vc, slots.view(1, 2), 64)
    with pytest.raises(ValueError, match="dense 4-bit"):
        ops.read_kv_int4(kc, vc, slots, 128)
    meta = _meta([1, 1], [1, 1], torch.zeros(2, 1, dtype=torch.int32), 4, 2, 64)
    q = torch.zeros(2, 4, 64)
    for kw, why in ((dict(q=q[:, :3]), "evenly"), (dict(q=q[0]), "queries"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
                    (dict(scale=float("nan")), "scale"), (dict(window=-1), "window"), (dict(out=torch.zeros(2, 4, 32)), "out"),
                    (dict(out=q.double()), "out"), (dict(q=torch.zeros(2, 4, 96)), "takes heads")):
        with pytest.raises(ValueError, match=why):
            ops.paged_attention_int4(**{**dict(q=q, k_cache=kc, v_cache=vc, meta=meta, scale=0.125), **kw})
    for kw in (dict(seq_lens=meta.seq_lens.long()), dict(block_table=meta.block_table[:1]), dict(query_start_loc=meta.query_start_loc[:2])):
        with pytest.raises(ValueError, match="metadata of 2 sequences"):
            ops.paged_attention_int4(q, kc, vc, dataclasses.replace(meta, **kw), 0.125)


def test_which_sequences_share_a_launch():
    from vllm_ascend_b200.ops.kv_int4 import _plan
    cu = np.cumsum([0, 1, 8, 9, 1, 0, 300, 2]).astype(np.int32).tobytes()
    def plan(cu, lens, G, fixed=False, window=0):
        return _plan(cu, "i", np.array(lens + [7], dtype=np.int64).tobytes(), "l", len(lens), window, G, 8, 128, 148, fixed)
    lens = [5000] * 7
    assert plan(cu, lens, 4) == ((True, 0, 2, (8,)), (False, 2, 7, (312, 8)))
    assert plan(cu, lens, 4, True) == ((True, 0, 2, (8,)), (False, 2, 3, (9, 1)), (True, 3, 5, (1,)), (False, 5, 6, (300, 5)), (True, 6, 7, (2,)))
    assert plan(cu, lens, 128) == ((False, 0, 7, (321, 162)),)
    assert plan(np.array([0, 1, 3], dtype=np.int32).tobytes(), [9, 9], 4) == ((True, 0, 2, (2,)),)
    # what lies behind the first ones may take less time in that kernel too: all in one launch, unless that leaves most of its blocks idle
    short = np.array([0, 1, 2, 40], dtype=np.int32).tobytes()
    assert plan(short, [600, 500, 38], 4) == ((True, 0, 3, (38,)),)
    assert plan(short, [600, 500, 38], 4, True) == ((True, 0, 2, (1,)), (False, 2, 3, (38, 1)))
    many = np.concatenate([np.arange(201), [300]]).astype(np.int32).tobytes()
    assert plan(many, [600] * 200 + [100], 4) == ((True, 0, 200, (1,)), (True, 200, 201, (100,)))
    assert plan(many, [600] * 200 + [0], 4, window=10)[0] == (True, 0, 200, (1,))


def test_parts_of_few_rows():
    from vllm_ascend_b200.ops.kv_int4 import _parts, _parts_of_rounds
    assert [_parts(8, n, 444, True) for n in (0, 100, 1000, 7000, 12000, 40001)] == [1, 1, 8, 8, 16, 18]
    assert [_parts(8, n, 444, False) for n in (30000, 40001)] == [8, 16]          # a graph's table
    assert [_parts(b, 20000, 444, True) for b in (24, 25, 32, 44)] == [14, 8, 8, 8]
    assert [_parts(b, 8000, 444, True) for b in (100, 222, 300)] == [4, 2, 1]
    assert [_parts_of_rounds(b, 11000, 8000.0, 444, 128) for b in (240, 2048)] == [4, 1]
    assert all(1 <= _parts_of_rounds(b, n, n / 2, 444, D) <= 8 for b in (223, 444, 10 ** 6) for n in (2048, 10 ** 6) for D in (64, 128))


def test_nothing_to_do():
    kc, vc = (ops.alloc_kv_cache_int4(2, 16, 2, 64, "cpu") for _ in "kv")
    none = torch.zeros(0, dtype=torch.int64)
    ops.write_kv_int4(torch.zeros(0, 2, 64), torch.zeros(0, 2, 64), kc, vc, none)
    assert ops.read_kv_int4(kc, vc, none, 64)[0].shape == (0, 2, 64)
    x = torch.ones(3, 2, 64, dtype=torch.bfloat16)
    ops.write_kv_int4(x, x, kc, vc, torch.full((3,), -1))
    assert not kc.any() and not vc.any()
    k, v = ops.read_kv_int4(kc, vc, torch.tensor([0, -1, 31]), 64)
    assert not k.any() and not v.any()             # a fresh cache stands for zeros
