"""Selection over beams and vocabulary, and reordering of beams' states, on the GPU."""
import math

import pytest
import torch

from beam_cases import check_select, reorder

pytestmark = pytest.mark.gpu


def _ops():
    from vllm_ascend_b200 import ops
    return ops


def _logits(rows, vocab, seed=0, dtype=torch.bfloat16, std=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty((rows, vocab), device="cuda").normal_(std=std, generator=g)
    hot = torch.randint(0, vocab, (rows, 5), generator=g, device="cuda")
    x.scatter_add_(1, hot, torch.empty((rows, 5), device="cuda").uniform_(2, 10, generator=g))
    return x.to(dtype)


def _scores(groups, width, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return -torch.empty((groups, width), device="cuda").exponential_(generator=g) * 4


SIZES = [(1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 7, 21), (1, 4, 32000, 8), (3, 5, 50257, 10), (7, 2, 4097, 4), (2, 8, 151936, 16), (1, 64, 6151, 128),
         (2, 16, 20011, 256), (1, 1, 300000, 256), (40, 8, 32000, 16), (1, 200, 999, 100), (700, 1, 8191, 3), (1, 1, 4096, 64), (1, 2, 8192, 33)]


@pytest.mark.parametrize("groups,width,vocab,k", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_best_continuations(groups, width, vocab, k, dtype):
    logits, scores = _logits(groups * width, vocab, vocab, dtype), _scores(groups, width)
    check_select(_ops().beam_select(logits, scores, k), logits, scores, k)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
def test_other_types(dtype):
    logits, scores = _logits(6, 1003, 3, dtype), _scores(2, 3)
    check_select(_ops().beam_select(logits, scores), logits.float(), scores, 6)


@pytest.mark.parametrize("vocab", [5, 131, 5000, 40001])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_without_candidates(vocab, dtype):
    logits, scores = _logits(12, vocab, 5, dtype), _scores(3, 4)
    logits[0] = -math.inf
    logits[1, vocab // 2] = math.nan
    logits[2, vocab - 1] = math.inf
    scores[0, 3], scores[1, 0], scores[1, 2] = -math.inf, math.nan, math.inf
    logits[7] = -math.inf
    logits[7, vocab // 3] = 1.5                                     # one candidate
    logits[8:, 1:] = -math.inf                                      # fewer than asked for
    k = min(9, 4 * vocab)
    got = _ops().beam_select(logits, scores, k)
    check_select(got, logits, scores, k)
    assert got[0][2, 4:].eq(-math.inf).all()


def test_ended_beams_are_not_read():
    logits, scores = _logits(8, 9001, 6), _scores(2, 4)
    logits[2], scores[0, 2] = math.nan, -math.inf
    check_select(_ops().beam_select(logits, scores, 8), logits, scores, 8)


@pytest.mark.parametrize("k", [1, 4, 16, 100, 256])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two", "steps", "zeros", "late"])
def test_orders_and_ties(kind, k):
    v = 30011
    at = torch.arange(v, device="cuda")
    row = {"equal": torch.full((v,), 0.5, device="cuda"), "rising": at / 1000.0, "falling": -at / 1000.0, "two": (at % 2).float(),
           "steps": (at // 5000).float(), "zeros": torch.where(at % 3 == 0, 0.0, -0.0), "late": (at >= v - 5000).float() * 3}[kind]
    logits = torch.stack([row, row - 0.25, row.flip(0)])
    scores = torch.tensor([[-1.0, -1.0, -2.5]], device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        x = logits.to(dtype)
        check_select(_ops().beam_select(x, scores, k), x, scores, k)


def test_equal_beams_come_in_order():
    logits = _logits(1, 20000, 8).expand(6, -1).contiguous()
    scores = torch.full((1, 6), -2.0, device="cuda")
    values, parents, tokens = _ops().beam_select(logits, scores, 12)
    check_select((values, parents, tokens), logits, scores, 12)
    assert parents[0].tolist()[:6] == list(range(6)) and len(set(tokens[0].tolist()[:6])) == 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad,first", [(0, 1), (3, 0), (5, 3), (8, 0), (1, 7)])
def test_strides_and_alignment(dtype, pad, first):
    whole = _logits(6, 10007 + pad + first, 9, dtype)
    logits, scores = whole[:, first:first + 10007], _scores(2, 3)
    check_select(_ops().beam_select(logits, scores, 6), logits, scores, 6)
    turned = logits.t().contiguous().t()
    check_select(_ops().beam_select(turned, scores.t().contiguous().t(), 6), logits, scores, 6)


def test_rows_repeat_bit_for_bit_and_groups_do_not_matter():
    logits, scores = _logits(24, 33333, 10), _scores(6, 4)
    a = _ops().beam_select(logits, scores, 8)
    b = _ops().beam_select(logits, scores, 8)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_no_groups():
    out = _ops().beam_select(torch.empty((0, 100), device="cuda"), torch.empty((0, 4), device="cuda"), 8)
    assert [tuple(t.shape) for t in out] == [(0, 8)] * 3


def test_two_streams_and_a_graph():
    ops = _ops()
    sets = [(_logits(16, 50021, s), _scores(4, 4, s)) for s in (11, 12)]
    want = [ops.beam_select(*x, 8) for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for x, s in zip(sets, streams):
            with torch.cuda.stream(s):
                got.append(ops.beam_select(*x, 8))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    logits, scores = sets[0][0].clone(), sets[0][1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.beam_select(logits, scores, 8)
    for x, w in zip(sets, want):
        logits.copy_(x[0])
        scores.copy_(x[1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, w))


# ---------------------------------------------------------------- reordering
def _rows(groups, width, held, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(held, generator=g)[:groups * width].int().view(groups, width)


def _parents(groups, width, seed=0):
    g = torch.Generator().manual_seed(seed + 100)
    return torch.randint(0, width, (groups, width), generator=g).int()


def _same(tensors, want):
    for t, w in zip(tensors, want):
        assert torch.equal(t.cpu(), w), (t.shape, t.dtype)


@pytest.mark.parametrize("groups,width", [(1, 1), (1, 2), (3, 4), (2, 5), (5, 8), (2, 13), (3, 16), (2, 17), (1, 64), (1, 130), (1, 300), (1, 600),
                                          (1, 1024), (70, 3)])
def test_states_follow_their_parents(groups, width):
    held = groups * width + 2
    shapes = [((held, 6, 16, 8), torch.float32), ((held, 24, 3), torch.bfloat16), ((held, 5), torch.uint8), ((held,), torch.int64),
              ((held, 3), torch.float16), ((held, 7, 2), torch.int32), ((held, 1031), torch.float32)]
    g = torch.Generator().manual_seed(width)
    host = [torch.randint(0, 100, s, generator=g).to(t) for s, t in shapes]
    rows, parents = _rows(groups, width, held, width), _parents(groups, width, width)
    want = reorder(host, rows, parents)
    dev = [t.cuda() for t in host]
    _ops().reorder_beams(_ops().beam_states(dev), rows.cuda(), parents.cuda())
    _same(dev, want)


@pytest.mark.parametrize("parents", [[1, 2, 3, 0], [1, 0, 3, 2], [0, 1, 2, 3], [3, 3, 3, 3], [-1, 0, -1, 2], [2, 2, 2, -1]])
def test_cycles_and_beams_that_stay(parents):
    x = torch.randn(9, 300)
    rows, p = torch.tensor([[7, 2, 4, 0]], dtype=torch.int32), torch.tensor([parents], dtype=torch.int32)
    want = reorder([x], rows, p)
    dev = [x.cuda()]
    _ops().reorder_beams(_ops().beam_states(dev), rows.cuda(), p.cuda())
    _same(dev, want)


def test_groups_of_fewer_beams():
    x = torch.randn(12, 40)
    rows = torch.tensor([[3, 1, 5], [0, -1, -1], [7, 11, -1]], dtype=torch.int32)
    p = torch.tensor([[1, 1, 0], [0, 0, 0], [1, 0, -1]], dtype=torch.int32)
    want = reorder([x], rows, p)
    dev = [x.cuda()]
    _ops().reorder_beams(_ops().beam_states(dev), rows.cuda(), p.cuda())
    _same(dev, want)


@pytest.mark.parametrize("order", ["tokens", "heads"])
@pytest.mark.parametrize("heads,dim,page,dtype", [(8, 128, 128, torch.bfloat16), (1, 64, 16, torch.bfloat16), (3, 40, 32, torch.float32),
                                                  (2, 7, 16, torch.float16), (1, 576, 64, torch.bfloat16)])
def test_pages_as_far_as_they_are_filled(order, heads, dim, page, dtype):
    groups, width = 5, 6
    held = groups * width + 3
    g = torch.Generator().manual_seed(dim)
    host = [torch.randn(held, page, heads, dim, generator=g).to(dtype) for _ in range(3)]
    if order == "heads":
        host = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in host]
    lengths = torch.tensor([0, 1, page // 2 + 1, page, page + 9], dtype=torch.int32)
    rows, parents = _rows(groups, width, held), _parents(groups, width)
    want = reorder(host, rows, parents, lengths)
    dev = [t.cuda() for t in host]
    states = _ops().beam_states(dev, paged=True)
    _ops().reorder_beams(states, rows.cuda(), parents.cuda(), lengths.cuda())
    _same(dev, want)
    _ops().reorder_beams(states, rows.cuda(), parents.cuda())               # whole pages
    _same(dev, reorder(want, rows, parents))


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 128)])
def test_pages_of_four_bits(dim, page):
    groups, width, heads = 3, 4, 5
    held = groups * width + 1
    g = torch.Generator().manual_seed(dim)
    host = [torch.randint(0, 256, (held, heads, page // 16 * 9 * dim), generator=g, dtype=torch.uint8) for _ in range(2)]
    lengths = torch.tensor([1, 16, 5], dtype=torch.int32)
    rows, parents = _rows(groups, width, held), _parents(groups, width)
    want = reorder(host, rows, parents, lengths, 9 * dim)
    dev = [t.cuda() for t in host]
    _ops().reorder_beams(_ops().beam_states(dev, paged=True, int4_dim=dim), rows.cuda(), parents.cuda(), lengths.cuda())
    _same(dev, want)


def test_views_of_larger_tensors():
    whole = torch.randn(20, 8, 50)
    dev = whole.cuda()
    views = [dev[:, 1], dev[:, 3, :48], dev[::2, 5], dev[3:13, 7, 1:48]]
    rows, parents = _rows(2, 4, 10), _parents(2, 4)
    want = whole.clone()
    for i, v in enumerate([want[:, 1], want[:, 3, :48], want[::2, 5], want[3:13, 7, 1:48]]):
        v.copy_(reorder([v], rows, parents)[0])
    _ops().reorder_beams(_ops().beam_states(views), rows.cuda(), parents.cuda())
    assert torch.equal(dev.cpu(), want)


def test_rows_and_parents_out_of_range_are_reported():
    from vllm_ascend_b200 import _native
    x = torch.randn(6, 64)
    for rows, parents in (([0, 1, 9], [1, 0, 0]), ([0, 1, -7], [1, 0, 0]), ([0, 1, 2], [1, 0, 3]), ([0, 1, 2], [1, 0, -5]), ([0, -1, 2], [0, 0, 1])):
        dev = x.cuda()
        _ops().reorder_beams(_ops().beam_states([dev]), torch.tensor([rows], dtype=torch.int32).cuda(),
                             torch.tensor([parents], dtype=torch.int32).cuda())
        torch.cuda.synchronize()
        with pytest.raises(_native.NativeError, match="BAD_INDEX"):
            _native.check_status(dev.device)
        if rows == [0, 1, 2]:
            assert torch.equal(dev.cpu(), reorder([x], torch.tensor([[0, 1]]), torch.tensor([[1, 0]]))[0])      # the others moved


def test_a_row_of_more_than_four_gigabytes():
    """Offsets past 32 bits: a tensor of 3 rows of 2.2 GB in bytes."""
    x = torch.zeros((3, 2_200_000_016), dtype=torch.uint8, device="cuda")
    x[0, :16], x[0, -16:], x[2, -16:] = 7, 9, 5
    rows, parents = torch.tensor([[0, 2]], dtype=torch.int32).cuda(), torch.tensor([[1, 0]], dtype=torch.int32).cuda()
    _ops().reorder_beams(_ops().beam_states([x]), rows, parents)
    assert x[2, :16].eq(7).all() and x[2, -16:].eq(9).all() and x[0, -16:].eq(5).all() and x[0, :16].eq(0).all() and not x[1].any()


def test_reordering_in_a_graph_follows_a_selection():
    ops = _ops()
    logits, scores = _logits(8, 3001, 20), _scores(2, 4)
    state = torch.randn(8, 500, device="cuda")
    rows = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    handle = ops.beam_states([state])

    def step():
        totals, parents, tokens = ops.beam_select(logits, scores, 8)
        ops.reorder_beams(handle, rows, parents[:, :4])
        return parents
    start = state.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        parents = step()
    for seed in (21, 22):
        logits.copy_(_logits(8, 3001, seed))
        state.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        want = reorder([start.cpu()], rows.cpu(), parents[:, :4].cpu())
        assert torch.equal(state.cpu(), want[0])
