"""Batches whose sequences share prefixes, their attention in 64 bits, and what a kernel may be off by."""
import numpy as np
import torch

from vllm_ascend_b200.attention.metadata import metadata_from_tensors


class Batch:
    """groups: [(prefix length, [(own tokens, new ones included, new tokens), ..])]; sequences of ``alone`` ahead of all groups.

    Pages hold NaN wherever no key of a sequence lies, tables page numbers out of range behind a sequence's last page and, for all but the first
    sequence of a group, in place of the prefix's whole pages."""

    def __init__(self, groups, heads, kv_heads, dim, page, alone=(), seed=0, device="cpu", dtype=torch.bfloat16, order="heads", pad_rows=0, std=1.0):
        g = torch.Generator().manual_seed(seed)
        groups = [(0, [s]) for s in alone] + list(groups)
        n = sum(len(s) for _, s in groups)
        lens = [p + own for p, seqs in groups for own, _ in seqs]
        new = [k for _, seqs in groups for _, k in seqs]
        total = sum(-(-x // page) for x in lens) + 4
        self.k = torch.full((total, page, kv_heads, dim), float("nan"), dtype=torch.float32)
        self.v = self.k.clone()
        ids = torch.randperm(total, generator=g).tolist()
        junk = 10 ** 6
        self.table = torch.full((n, max(1, max((-(-x // page) for x in lens), default=1)) + 2), junk, dtype=torch.int32)
        self.keys, self.values, s = [], [], 0            # of every sequence, dense
        starts, prefixes = [], []
        for prefix, seqs in groups:
            starts.append(s)
            prefixes.append(prefix)
            pages = [ids.pop() for _ in range(-(-prefix // page))]
            kp, vp = torch.randn(prefix, kv_heads, dim, generator=g) * std, torch.randn(prefix, kv_heads, dim, generator=g)
            kp, vp = kp.to(dtype).float(), vp.to(dtype).float()
            for i, (own, _) in enumerate(seqs):
                mine = []
                for c in range(-(-(prefix + own) // page)):
                    whole = (c + 1) * page <= prefix
                    if i == 0 and c < len(pages):
                        self.table[s, c] = pages[c]
                    elif not whole:
                        self.table[s, c] = ids.pop()
                    mine.append(int(self.table[s, c]))
                ko, vo = torch.randn(own, kv_heads, dim, generator=g) * std, torch.randn(own, kv_heads, dim, generator=g)
                ko, vo = ko.to(dtype).float(), vo.to(dtype).float()
                for pos in range(prefix + own):
                    if pos < prefix and i > 0:
                        continue
                    self.k[mine[pos // page], pos % page] = kp[pos] if pos < prefix else ko[pos - prefix]
                    self.v[mine[pos // page], pos % page] = vp[pos] if pos < prefix else vo[pos - prefix]
                self.keys.append(torch.cat((kp, ko)))
                self.values.append(torch.cat((vp, vo)))
                s += 1
        first = len(alone)                               # the ones alone are in no group
        self.starts = torch.tensor(starts[first:] + [n], dtype=torch.int32)
        self.prefixes = torch.tensor(prefixes[first:], dtype=torch.int32)
        self.lens, self.new = lens, new
        self.rows = sum(new)
        whole = torch.randn(self.rows + pad_rows, heads + 2 * kv_heads, dim, generator=g).to(dtype)
        self.q = whole.to(device)[:, :heads]
        self.heads, self.kv_heads, self.dim, self.page, self.device = heads, kv_heads, dim, page, device
        self.scale = dim ** -0.5

        def cache(t):
            t = t.to(dtype)
            if order == "heads":
                t = t.transpose(1, 2).contiguous().transpose(1, 2)
            t = t.to(device)
            return t
        self.k_cache, self.v_cache = cache(self.k), cache(self.v)
        cu = torch.tensor(np.cumsum([0] + new), dtype=torch.int32)
        self.cu = cu
        self.meta = metadata_from_tensors(cu.to(device), torch.tensor(lens, dtype=torch.int32).to(device), self.table.to(device),
                                          max(new, default=0), max(lens, default=0), heads, kv_heads, dim)
        self.starts, self.prefixes = self.starts.to(device), self.prefixes.to(device)

    def plan(self, ops):
        return ops.plan_shared_prefix(self.meta, self.starts, self.prefixes, self.heads, self.kv_heads)

    def run(self, ops, out=None):
        return ops.paged_attention_shared(self.q, self.k_cache, self.v_cache, self.meta, self.plan(ops), self.scale, out)

    def exact(self):
        """Results and what they may be off by, in 64 bits.  A result rounds to its type (half a step, e); probabilities round to bf16 in front of
        their product (2^-8 of what each adds); scores are sums of ``dim`` products in fp32 (half a step each, of their magnitudes), exponentials are
        off by 2 ulp."""
        q, per = self.q.double().cpu(), self.heads // self.kv_heads
        outs, offs, at = [], [], 0
        e = torch.finfo(self.q.dtype).eps / 2
        for k, v, n, new in zip(self.keys, self.values, self.lens, self.new):
            rows = q[at:at + new].unflatten(1, (self.kv_heads, per))
            k, v = k.double(), v.double()
            s = torch.einsum("tghd,kgd->ghtk", rows, k) * self.scale
            size = torch.einsum("tghd,kgd->ghtk", rows.abs(), k.abs()) * self.scale
            seen = torch.arange(n)[None] <= torch.arange(n - new, n)[:, None]
            s, size = torch.where(seen, s, -torch.inf), torch.where(seen, size, 0.0)
            p = torch.where(seen.any(-1)[None, None, :, None], torch.softmax(s, -1), 0.0)
            o = torch.einsum("ghtk,kgd->tghd", p, v).flatten(1, 2)
            spread = torch.einsum("ghtk,kgd->tghd", p, v.abs()).flatten(1, 2)
            off = 2 * (self.dim + 2) * 2.0 ** -24 * float(size.max() if size.numel() else 0.0) + 2.0 ** -20
            outs.append(o)
            offs.append(e * o.abs() + (2.0 ** -8 + off) * spread + 1e-30)
            at += new
        if not outs:
            return torch.zeros_like(q), torch.zeros_like(q)
        return torch.cat(outs), torch.cat(offs)

    def check(self, out):
        want, off = self.exact()
        got = out[:self.rows].double().cpu()
        assert got.isfinite().all()
        wrong = (got - want).abs() > off
        assert not wrong.any(), f"{int(wrong.sum())} of {wrong.numel()}, worst {float(((got - want).abs() / off).max()):.2f} of what it may be"
