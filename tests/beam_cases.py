"""Plain definitions in 64 bits of the steps of a beam search, and what results may be off by."""
import math

import torch


def totals(logits, scores):
    """[groups, beams * vocab] in 64 bits; -inf where there is no candidate."""
    x = logits.double().cpu()
    lp = x - torch.logsumexp(x, -1, keepdim=True)
    total = scores.double().cpu().reshape(-1, 1) + lp
    total = torch.where(total.isfinite(), total, -math.inf)
    return total.view(scores.shape[0], -1)


def select(logits, scores, k):
    total = totals(logits, scores)
    best, at = torch.sort(total, dim=-1, descending=True, stable=True)
    v = logits.shape[1]
    return best[:, :k], at[:, :k] // v, at[:, :k] % v


def slack(logits):
    """What a total may be off by in front of its rounding to fp32: the sum's terms are off by 2 ulp of an exponential (2^-22), the rounding of
    the difference and its product with log2 e (2^-23 of |d| e^-|d|, below 2^-24), and a thread adds its terms (an eighth of a row's at most
    512th part, four sums side by side) in fp32, half a step each."""
    terms = logits.shape[1] / 512 + 8
    return 2.0 ** -22 + 2.0 ** -24 + terms * 2.0 ** -24


def check_select(got, logits, scores, k):
    """Totals to their rounding; places equal wherever neighbouring totals are further apart than what they may be off by."""
    values, parents, tokens = (t.cpu() for t in got)
    total, v = totals(logits, scores), logits.shape[1]
    best, beam, token = select(logits, scores, k)
    off = slack(logits)
    assert values.dtype == torch.float32 and parents.dtype == torch.int32 and tokens.dtype == torch.int64
    assert values.shape == parents.shape == tokens.shape == (scores.shape[0], k)
    finite = best.isfinite()
    assert torch.equal(values.isfinite(), finite)
    wrong = (values.double() - best).abs()[finite] > off + 2.0 ** -24 * best.abs()[finite] + 2.0 ** -24 * off
    assert not wrong.any()
    flat = parents.long() * v + tokens
    assert all(len(set(row.tolist())) == k for row in flat)
    mine = total.gather(1, flat)
    # what was taken is as good as the best, place by place, to twice the slack
    assert torch.equal(mine.isfinite(), finite)
    assert ((mine - best).abs()[finite] <= 2 * off).all()
    exact = beam * v + token
    order = torch.sort(total, dim=-1, descending=True, stable=True)[0]
    order = torch.cat((order, torch.full_like(order[:, :1], -math.inf)), 1)
    near = order[:, :k] - order[:, 1:k + 1]
    gap = torch.where(near.isnan(), 0.0, near)                            # -inf beside -inf: a tie
    gap[:, 1:] = torch.minimum(gap[:, 1:], gap[:, :-1].clone())
    told = (gap > 2 * off) | (gap == 0)
    same_row_tie = gap == 0                                               # equal totals: lowest place first, exactly
    assert torch.equal(flat[told & ~same_row_tie], exact[told & ~same_row_tie])
    assert torch.equal(flat[~finite], exact[~finite])
    # ties inside a beam come in the order of tokens
    for r in range(k - 1):
        tie = (mine[:, r] == mine[:, r + 1]) & (parents[:, r] == parents[:, r + 1])
        assert (flat[:, r][tie] < flat[:, r + 1][tie]).all()


def reorder(tensors, rows, parents, lengths=None, unit=1):
    """What ``tensors`` become; ``unit``: tokens that a page of 4 bits is copied in."""
    out = [t.clone() for t in tensors]
    for g in range(rows.shape[0]):
        for w in range(rows.shape[1]):
            p, row = int(parents[g, w]), int(rows[g, w])
            if p < 0 or row < 0:
                continue
            src = int(rows[g, p])
            for t, o in zip(tensors, out):
                if lengths is None:
                    o[row] = t[src]
                elif t.dtype == torch.uint8:
                    n = -(-int(lengths[g]) // 16) * unit
                    o[row, :, :n] = t[src, :, :n]
                else:
                    o[row, :int(lengths[g])] = t[src, :int(lengths[g])]
    return out
