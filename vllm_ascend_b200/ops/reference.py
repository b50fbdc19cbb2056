"""Plain PyTorch restatements of every op.

They are (a) the execution path for CPU tensors (the tiny fp32 correctness
config runs entirely through them) and (b) the fp32 oracle the GPU kernel tests
compare against — the same role numpy goldens play in the reference's op tests
(tests/e2e/nightly/single_node/ops/singlecard_ops/*).
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn.functional as F


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float,
             residual: Optional[torch.Tensor] = None, gemma: bool = False):
    orig = x.dtype
    if residual is not None:
        z = (x.float() + residual.float()).to(orig)
        residual = z
        xf = z.float()
    else:
        xf = x.float()
    var = xf.pow(2).mean(dim=-1, keepdim=True)
    w = weight.float() + 1.0 if gemma else weight.float()
    out = (xf * torch.rsqrt(var + eps) * w).to(orig)
    return out, residual


def silu_and_mul(x: torch.Tensor, limit: float = 0.0) -> torch.Tensor:
    d = x.shape[-1] // 2
    g, u = x[..., :d].float(), x[..., d:].float()
    if limit > 0:
        g = g.clamp(max=limit)
        u = u.clamp(min=-limit, max=limit)
    return (F.silu(g) * u).to(x.dtype)


def embedding(ids: torch.Tensor, weight: torch.Tensor, vocab_start: int = 0,
              vocab_end: Optional[int] = None) -> torch.Tensor:
    if vocab_end is None:
        vocab_end = vocab_start + weight.shape[0]
    mask = (ids >= vocab_start) & (ids < vocab_end)
    local = torch.where(mask, ids - vocab_start, torch.zeros_like(ids))
    out = F.embedding(local, weight)
    return out * mask.unsqueeze(-1).to(out.dtype)


def build_cos_sin_cache(rot_dim: int, max_pos: int, theta: float,
                        rope_scaling: Optional[dict] = None,
                        device="cpu") -> torch.Tensor:
    """fp32 [max_pos, rot_dim]: cos in the first half, sin in the second.

    Supports plain RoPE, linear and YaRN scaling (the variants of
    vllm_ascend/ops/rotary_embedding.py:233-578 that change only the table).
    """
    half = rot_dim // 2
    inv_freq = 1.0 / (theta ** (torch.arange(0, half, dtype=torch.float64) * 2 / rot_dim))
    mscale = 1.0
    if rope_scaling:
        kind = rope_scaling.get("rope_type", rope_scaling.get("type", "default"))
        factor = float(rope_scaling.get("factor", 1.0))
        if kind == "linear":
            inv_freq = inv_freq / factor
        elif kind in ("yarn", "deepseek_yarn", "yarn_interp"):
            orig = rope_scaling.get("original_max_position_embeddings", max_pos)
            beta_fast = rope_scaling.get("beta_fast", 32)
            beta_slow = rope_scaling.get("beta_slow", 1)

            def corr_dim(n_rot):
                return (rot_dim * math.log(orig / (n_rot * 2 * math.pi))) / (2 * math.log(theta))

            low = max(math.floor(corr_dim(beta_fast)), 0)
            high = min(math.ceil(corr_dim(beta_slow)), rot_dim - 1)
            if kind == "yarn_interp":
                high = low + max(high - low, 0.001)
            elif low == high:
                high += 0.001
            ramp = ((torch.arange(half, dtype=torch.float64) - low) / (high - low)).clamp(0, 1)
            mask = 1 - ramp
            inv_freq = inv_freq / factor * (1 - mask) + inv_freq * mask

            def yarn_mscale(scale, m=1.0):
                return 1.0 if scale <= 1 else 0.1 * m * math.log(scale) + 1.0

            if kind == "deepseek_yarn":
                mscale = (yarn_mscale(factor, rope_scaling.get("mscale", 1.0)) /
                          yarn_mscale(factor, rope_scaling.get("mscale_all_dim", 0.0) or 1.0)
                          if rope_scaling.get("mscale_all_dim") else
                          yarn_mscale(factor, rope_scaling.get("mscale", 1.0)))
            elif kind == "yarn_interp":         # the factor on cos and sin, without a floor at 1
                mscale = 0.1 * math.log(factor) + 1.0
            else:
                mscale = yarn_mscale(factor)
        elif kind == "llama3":
            lo_f = rope_scaling.get("low_freq_factor", 1.0)
            hi_f = rope_scaling.get("high_freq_factor", 4.0)
            orig = rope_scaling.get("original_max_position_embeddings", 8192)
            wavelen = 2 * math.pi / inv_freq
            smooth = ((orig / wavelen) - lo_f) / (hi_f - lo_f)
            scaled = torch.where(wavelen > orig / lo_f, inv_freq / factor, inv_freq)
            mid = (1 - smooth) * inv_freq / factor + smooth * inv_freq
            is_mid = (wavelen <= orig / lo_f) & (wavelen >= orig / hi_f)
            inv_freq = torch.where(is_mid, mid, scaled)
    t = torch.arange(max_pos, dtype=torch.float64)
    freqs = torch.outer(t, inv_freq)
    cache = torch.cat([freqs.cos() * mscale, freqs.sin() * mscale], dim=-1)
    return cache.float().to(device)


def apply_rope_neox(x: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                    rot_dim: int) -> torch.Tensor:
    """x: [T, H, D]; rotates the first rot_dim dims pairing j with j + rot_dim/2."""
    half = rot_dim // 2
    cs = cos_sin[positions]                       # [T, rot_dim]
    cos, sin = cs[:, :half].unsqueeze(1), cs[:, half:].unsqueeze(1)
    xf = x.float()
    x1, x2 = xf[..., :half], xf[..., half:rot_dim]
    out = xf.clone()
    out[..., :half] = x1 * cos - x2 * sin
    out[..., half:rot_dim] = x2 * cos + x1 * sin
    return out.to(x.dtype)


def mrope_axis_table(sections, interleaved: bool = False) -> torch.Tensor:
    """int32 [sum(sections)]: which position axis (0 temporal, 1 height, 2 width) each rotary
    pair follows.  Sectioned layout: the first sections[0] pairs are temporal, then height, then
    width (Qwen2-VL); interleaved layout: t h w t h w ... with the temporal axis taking what is
    left once height / width are used up (Qwen3-VL).  Follows the index arithmetic of
    vllm_ascend/ops/rotary_embedding.py:582-672 (the mrope paths)."""
    half = int(sum(sections))
    axis = torch.zeros(half, dtype=torch.int32)
    if interleaved:
        for a in (1, 2):
            idx = torch.arange(a, sections[a] * 3, 3)
            axis[idx[idx < half]] = a
    else:
        axis[sections[0]:sections[0] + sections[1]] = 1
        axis[sections[0] + sections[1]:] = 2
    return axis


def apply_mrope_neox(x: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                     rot_dim: int, axis: torch.Tensor) -> torch.Tensor:
    """x: [T, H, D]; positions int64 [3, >=T]; pair e rotates by the angle at positions[axis[e]]."""
    T = x.shape[0]
    half = rot_dim // 2
    pos = positions[:, :T][axis.long()]                      # [half, T]
    e = torch.arange(half, device=x.device).unsqueeze(1)
    cos = cos_sin[pos, e].t().unsqueeze(1)                   # [T, 1, half]
    sin = cos_sin[pos, e + half].t().unsqueeze(1)
    xf = x.float()
    x1, x2 = xf[..., :half], xf[..., half:rot_dim]
    out = xf.clone()
    out[..., :half] = x1 * cos - x2 * sin
    out[..., half:rot_dim] = x2 * cos + x1 * sin
    return out.to(x.dtype)


def apply_rope_interleaved(x: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                           rot_dim: int) -> torch.Tensor:
    """GPT-J style: pairs (2j, 2j+1); used by DeepSeek's rope slice."""
    half = rot_dim // 2
    cs = cos_sin[positions]
    cos, sin = cs[:, :half].unsqueeze(1), cs[:, half:].unsqueeze(1)
    xf = x.float()
    xr = xf[..., :rot_dim]
    x1, x2 = xr[..., 0::2], xr[..., 1::2]
    o1 = x1 * cos - x2 * sin
    o2 = x2 * cos + x1 * sin
    out = xf.clone()
    out[..., :rot_dim] = torch.stack([o1, o2], dim=-1).flatten(-2)
    return out.to(x.dtype)


def qknorm_rope_kvwrite(qkv: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                        rot_dim: int, q_norm_w, k_norm_w, eps: float,
                        k_cache: Optional[torch.Tensor], v_cache: Optional[torch.Tensor],
                        slot_mapping: Optional[torch.Tensor], Hq: int, Hkv: int, D: int,
                        mrope_axis: Optional[torch.Tensor] = None) -> None:
    """In place on qkv [T, (Hq+2Hkv)*D]; scatters k, v into the paged caches."""
    T = qkv.shape[0]
    q = qkv[:, :Hq * D].view(T, Hq, D)
    k = qkv[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D)
    v = qkv[:, (Hq + Hkv) * D:].view(T, Hkv, D)
    if q_norm_w is not None:
        q.copy_(rms_norm(q, q_norm_w, eps)[0])
    if k_norm_w is not None:
        k.copy_(rms_norm(k, k_norm_w, eps)[0])
    if rot_dim > 0 and mrope_axis is not None:
        q.copy_(apply_mrope_neox(q, positions, cos_sin, rot_dim, mrope_axis))
        k.copy_(apply_mrope_neox(k, positions, cos_sin, rot_dim, mrope_axis))
    elif rot_dim > 0:
        q.copy_(apply_rope_neox(q, positions, cos_sin, rot_dim))
        k.copy_(apply_rope_neox(k, positions, cos_sin, rot_dim))
    if k_cache is not None and slot_mapping is not None:
        valid = slot_mapping >= 0
        slots = slot_mapping[valid]
        bs = k_cache.shape[1]                      # works for any physical layout of the cache
        blk, off = slots // bs, slots % bs
        k_cache[blk, off] = k[valid].to(k_cache.dtype)
        v_cache[blk, off] = v[valid].to(v_cache.dtype)


def gather_kv(cache: torch.Tensor, block_table_row: torch.Tensor, seq_len: int) -> torch.Tensor:
    """cache [NB, BS, H, D] -> [seq_len, H, D] for one sequence."""
    bs = cache.shape[1]
    nblk = (seq_len + bs - 1) // bs
    blocks = block_table_row[:nblk].long()
    return cache[blocks].reshape(nblk * bs, *cache.shape[2:])[:seq_len]


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    query_start_loc, seq_lens, block_table: torch.Tensor, scale: float,
                    causal: bool = True, window: int = 0,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """q: [T, Hq, D]; every query attends to keys [0, ctx + own_pos] of its sequence."""
    T, Hq, D = q.shape
    Hkv = k_cache.shape[2]
    Dv = v_cache.shape[3]
    G = Hq // Hkv
    if out is None:
        out = torch.empty(T, Hq, Dv, dtype=q.dtype, device=q.device)
    lse_out = torch.full((T, Hq), float("-inf"), dtype=torch.float32, device=q.device)
    qsl = [int(x) for x in query_start_loc]
    sls = [int(x) for x in seq_lens]
    for b in range(len(sls)):
        qs, qe = qsl[b], qsl[b + 1]
        ql = qe - qs
        if ql <= 0:
            continue
        sl = sls[b]
        ctx = sl - ql
        k = gather_kv(k_cache, block_table[b], sl).float()       # [sl, Hkv, D]
        v = gather_kv(v_cache, block_table[b], sl).float()
        qq = q[qs:qe].float()                                     # [ql, Hq, D]
        k = k.repeat_interleave(G, dim=1)
        v = v.repeat_interleave(G, dim=1)
        s = torch.einsum("qhd,khd->hqk", qq, k) * scale
        kpos = torch.arange(sl, device=q.device)
        qpos = ctx + torch.arange(ql, device=q.device)
        mask = torch.ones(ql, sl, dtype=torch.bool, device=q.device)
        if causal:
            mask &= kpos[None, :] <= qpos[:, None]
        if window and window > 0:
            mask &= kpos[None, :] > (qpos[:, None] - window)
        s = s.masked_fill(~mask[None], float("-inf"))
        lse = torch.logsumexp(s, dim=-1)                          # [Hq, ql]
        p = torch.exp(s - lse.unsqueeze(-1))
        p = torch.nan_to_num(p, nan=0.0)
        o = torch.einsum("hqk,khd->qhd", p, v)
        out[qs:qe] = o.to(out.dtype)
        lse_out[qs:qe] = lse.transpose(0, 1)
    if return_lse:
        return out, lse_out
    return out


# ---------------------------------------------------------------- 4-bit cache
KV_INT4_GROUP, KV_INT4_TOKENS = 32, 16


def kv_int4_quantise(x: torch.Tensor):
    """x [..., D] -> whole numbers in -7..7 (int8) [..., D] and scales (bf16) [..., D / 32].  A scale is the smallest number
    of five significant bits with 7 scale >= max |x| over its 32 channels, between 2^-80 and 2^34 (larger magnitudes saturate), or zero
    for a group of zeros; a group that holds a NaN or an infinity is NaN."""
    g = x.float().unflatten(-1, (-1, KV_INT4_GROUP))
    top = g.abs().amax(-1, keepdim=True)
    finite = torch.isfinite(top)
    top = torch.where(finite, top, 0.0)
    low = top / torch.full_like(top, 7.0)
    s = ((low.view(torch.int32) + 0x7ffff) & ~0x7ffff).view(torch.float32).clamp(2.0 ** -80, 2.0 ** 34)
    s = torch.where(top > 0, s, 0.0)
    n = torch.where(finite & (s > 0), g / torch.where(s > 0, s, 1.0), 0.0).clamp(-7, 7).round()
    nan = torch.tensor(0x7fc0, dtype=torch.int16, device=x.device).view(torch.bfloat16)      # the same bits everywhere
    s = torch.where(finite, s.to(torch.bfloat16), nan)
    return n.flatten(-2).to(torch.int8), s.squeeze(-1)


def kv_int4_block_size(cache: torch.Tensor, dim: int) -> int:
    """Tokens of a block of a 4-bit cache [blocks, heads, bytes]; raises where the bytes do not fit heads of ``dim``."""
    unit = 9 * dim
    if cache.dtype != torch.uint8 or cache.dim() != 3 or not cache.is_contiguous() or cache.shape[2] == 0 or cache.shape[2] % unit:
        raise ValueError(f"not a dense 4-bit cache [blocks, heads, bytes] of heads of {dim}: {cache.dtype} {tuple(cache.shape)}")
    return cache.shape[2] // unit * KV_INT4_TOKENS


def _kv_int4_views(cache: torch.Tensor, dim: int, values: bool):
    """Bytes and scales of a cache, [blocks, heads, units, ...] each (csrc/kv_int4.cuh has the layout).  Keys: [token, byte], values:
    [pair of tokens, chunk, word, token of the pair, byte]; scales [group, token]."""
    B, H, _ = cache.shape
    units = kv_int4_block_size(cache, dim) // KV_INT4_TOKENS
    data = cache.view(B, H, units, 9 * dim)[..., :8 * dim]
    scales = cache.view(torch.bfloat16).view(B, H, units, 9 * dim // 2)[..., 4 * dim:]
    data = data.unflatten(-1, (8, dim // 16, 4, 2, 2) if values else (KV_INT4_TOKENS, dim // 2))
    return data, scales.unflatten(-1, (dim // KV_INT4_GROUP, KV_INT4_TOKENS))


def _kv_int4_chunks(pair: torch.Tensor, dim: int) -> torch.Tensor:
    """Where chunk 0, 1, ... of a pair's values lie: [tokens, chunks]."""
    swizzle = 2 * (pair & 3) if dim == 128 else pair & 2
    return torch.arange(dim // 16, device=pair.device) ^ swizzle.unsqueeze(-1)


def write_kv_int4(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor) -> None:
    dim = k.shape[-1]
    bs = kv_int4_block_size(k_cache, dim)
    valid = slots >= 0
    at = slots[valid]
    blk, off = at // bs, at % bs
    unit, t = off // KV_INT4_TOKENS, off % KV_INT4_TOKENS
    heads = torch.arange(k.shape[1], device=k.device).view(1, -1, 1)
    for x, cache, values in ((k, k_cache, False), (v, v_cache, True)):
        data, scales = _kv_int4_views(cache, dim, values)
        n, s = kv_int4_quantise(x[valid])
        n = (n + 8).to(torch.uint8)
        n = n[..., 0::2] | (n[..., 1::2] << 4)                                   # bytes of two channels, in order
        if values:
            b, u, pair, half = (i.view(-1, 1, 1) for i in (blk, unit, t >> 1, t & 1))
            data[b, heads, u, pair, _kv_int4_chunks(t >> 1, dim).unsqueeze(1), :, half] = n.unflatten(-1, (dim // 16, 4, 2))
        else:
            data[blk, :, unit, t] = n
        scales[blk, :, unit, :, t] = s


def read_kv_int4(k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, dim: int, dtype=torch.bfloat16):
    bs = kv_int4_block_size(k_cache, dim)
    at = slots.clamp(min=0)
    blk, off = at // bs, at % bs
    unit, t = off // KV_INT4_TOKENS, off % KV_INT4_TOKENS
    out = []
    heads = torch.arange(k_cache.shape[1], device=slots.device).view(1, -1, 1)
    for cache, values in ((k_cache, False), (v_cache, True)):
        data, scales = _kv_int4_views(cache, dim, values)
        if values:
            b, u, pair, half = (i.view(-1, 1, 1) for i in (blk, unit, t >> 1, t & 1))
            w = data[b, heads, u, pair, _kv_int4_chunks(t >> 1, dim).unsqueeze(1), :, half].flatten(-3)
        else:
            w = data[blk, :, unit, t]
        s = scales[blk, :, unit, :, t]
        n = torch.stack((w & 15, w >> 4), -1).flatten(-2).float() - 8
        x = (n.unflatten(-1, (-1, KV_INT4_GROUP)) * s.float().unsqueeze(-1)).flatten(-2)
        out.append(torch.where((slots >= 0).view(-1, 1, 1), x, 0.0).to(dtype))
    return tuple(out)


def paged_attention_int4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, query_start_loc, seq_lens,
                         block_table: torch.Tensor, scale: float, causal: bool = True, window: int = 0, out: Optional[torch.Tensor] = None):
    dim = q.shape[-1]
    B, bs = k_cache.shape[0], kv_int4_block_size(k_cache, dim)
    k, v = read_kv_int4(k_cache, v_cache, torch.arange(B * bs, device=q.device), dim, torch.float32)
    odd_k, odd_v = k.isnan().any(-1), v.unflatten(-1, (-1, KV_INT4_GROUP)).isnan().any(-1)              # [slots, heads], with groups
    no_numbers = bool(odd_k.any() or odd_v.any())
    if no_numbers:
        k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
    out = paged_attention(q, *(t.view(B, bs, -1, dim) for t in (k, v)), query_start_loc, seq_lens, block_table, scale, causal, window, out=out)
    # groups that are no numbers reach the rows that see them, and no others
    for b in range(len(seq_lens) if no_numbers else 0):
        first, end, n = int(query_start_loc[b]), int(query_start_loc[b + 1]), int(seq_lens[b])
        if end <= first:
            continue
        pos = torch.arange(n, device=q.device)
        own, at = torch.arange(n - (end - first), n, device=q.device).unsqueeze(1), block_table[b].long()[pos // bs] * bs + pos % bs
        sees = torch.ones((end - first, n), dtype=torch.bool, device=q.device)
        if causal:
            sees &= pos <= own
        if window > 0:
            sees &= pos > own - window
        hit = (torch.einsum("qk,kh->qh", sees.float(), odd_k[at].float()) > 0).unsqueeze(-1) \
            | (torch.einsum("qk,khg->qhg", sees.float(), odd_v[at].float()) > 0)
        hit = hit.repeat_interleave(q.shape[1] // odd_k.shape[1], 1).repeat_interleave(KV_INT4_GROUP, 2)
        out[first:end] = torch.where(hit, float("nan"), out[first:end])
    return out


def merge_attn_states(o1, lse1, o2, lse2):
    """LSE merge of two partial attention results ([T,H,D], [T,H])."""
    m = torch.maximum(lse1, lse2)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    w1, w2 = torch.exp(lse1 - m), torch.exp(lse2 - m)
    den = (w1 + w2).clamp_min(1e-30)
    o = (o1.float() * (w1 / den).unsqueeze(-1) + o2.float() * (w2 / den).unsqueeze(-1))
    return o.to(o1.dtype), m + torch.log(den)


# ---------------------------------------------------------------- sampling
def apply_penalties(logits: torch.Tensor, prompt_ids: torch.Tensor, output_ids: torch.Tensor,
                    rep: torch.Tensor, freq: torch.Tensor, pres: torch.Tensor) -> torch.Tensor:
    """logits fp32 [B, V]; id tensors padded with values >= V."""
    B, V = logits.shape
    out_counts = torch.zeros(B, V + 1, dtype=torch.float32, device=logits.device)
    out_counts.scatter_add_(1, output_ids.clamp(min=0, max=V),
                            torch.ones_like(output_ids, dtype=torch.float32))
    out_counts = out_counts[:, :V]
    prompt_mask = torch.zeros(B, V + 1, dtype=torch.bool, device=logits.device)
    prompt_mask.scatter_(1, prompt_ids.clamp(min=0, max=V), True)
    seen = prompt_mask[:, :V] | (out_counts > 0)
    r = rep.unsqueeze(1)
    scaled = torch.where(logits > 0, logits / r, logits * r)
    logits = torch.where(seen, scaled, logits)
    logits = logits - freq.unsqueeze(1) * out_counts - pres.unsqueeze(1) * (out_counts > 0).float()
    return logits


def top_k_top_p_filter(probs: torch.Tensor, top_k: torch.Tensor, top_p: torch.Tensor,
                       min_p: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Sort-based reference: returns the filtered (unnormalised) probabilities."""
    B, V = probs.shape
    sp, si = probs.sort(dim=-1, descending=True)
    ranks = torch.arange(V, device=probs.device).unsqueeze(0)
    k = torch.where((top_k <= 0) | (top_k >= V), torch.full_like(top_k, V), top_k).unsqueeze(1)
    keep = ranks < k
    # ties with the k-th value stay (the radix select keeps them too)
    kth = sp.gather(1, (k - 1).clamp(min=0))
    keep |= sp >= kth
    spk = sp * keep
    mass = spk.sum(-1, keepdim=True)
    cum = spk.cumsum(-1)
    p = top_p.unsqueeze(1)
    keep_p = (cum - spk) < p * mass          # smallest prefix whose mass reaches p
    keep_p[:, 0] = True
    keep &= torch.where(p >= 1.0, torch.ones_like(keep_p), keep_p)
    if min_p is not None:
        keep &= sp >= (min_p.unsqueeze(1) * sp[:, :1])
    out = torch.zeros_like(probs)
    out.scatter_(1, si, sp * keep)
    return out


def sample(logits: torch.Tensor, temperature: torch.Tensor, top_k: torch.Tensor,
           top_p: torch.Tensor, min_p: Optional[torch.Tensor] = None,
           generator: Optional[torch.Generator] = None, seeds: Optional[torch.Tensor] = None,
           offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Greedy rows (temperature < 1e-5) take argmax; others the exponential race.  With ``seeds`` /
    ``offsets`` every row draws from its own stream (request seed, number of tokens generated so
    far), so a request's samples do not depend on what else is in the batch."""
    greedy = temperature < 1e-5
    t = torch.where(greedy, torch.ones_like(temperature), temperature).unsqueeze(1)
    probs = torch.softmax(logits.float() / t, dim=-1)
    probs = top_k_top_p_filter(probs, top_k, top_p, min_p)
    if seeds is not None:
        e = torch.empty_like(probs)
        off = offsets if offsets is not None else torch.zeros_like(seeds)
        for i in range(probs.shape[0]):
            g = torch.Generator(device="cpu").manual_seed((int(seeds[i]) * 1000003 + int(off[i])) & ((1 << 63) - 1))
            e[i].exponential_(1.0, generator=g)
    else:
        e = torch.empty_like(probs).exponential_(1.0, generator=generator)
    sampled = (probs / e).argmax(dim=-1)
    return torch.where(greedy, logits.argmax(dim=-1), sampled)


# ---------------------------------------------------------------- quantization
def quant_fp8_group128(x: torch.Tensor, pow2_scale: bool = False):
    """Per-token groups of 128 columns (the last group may be shorter)."""
    T, H = x.shape
    G = (H + 127) // 128
    xp = torch.zeros(T, G * 128, dtype=torch.float32, device=x.device)
    xp[:, :H] = x.float()
    xg = xp.view(T, G, 128)
    amax = xg.abs().amax(dim=-1).clamp_min(1e-10)
    scale = amax / 448.0
    if pow2_scale:
        scale = torch.exp2(torch.ceil(torch.log2(scale)))
    q = (xg / scale.unsqueeze(-1)).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q.view(T, G * 128)[:, :H].contiguous(), scale


def dequant_block_fp8_weight(w: torch.Tensor, scale: torch.Tensor, block=(128, 128)):
    N, K = w.shape
    bn, bk = block
    s = scale.repeat_interleave(bn, dim=0)[:N].repeat_interleave(bk, dim=1)[:, :K]
    return w.float() * s


def block_fp8_linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, block=(128, 128),
                     out_dtype=torch.bfloat16) -> torch.Tensor:
    xq, xs = quant_fp8_group128(x)
    K = x.shape[1]
    xd = xq.float() * xs.repeat_interleave(128, dim=1)[:, :K]
    wd = dequant_block_fp8_weight(w, w_scale, block)
    return (xd @ wd.t()).to(out_dtype)


# ---------------------------------------------------------------- more activations / gated norm
def quant_fp8_per_token(x: torch.Tensor):
    xf = x.float()
    scale = (xf.abs().amax(dim=-1) / 448.0).clamp_min(1e-10)
    return (xf / scale.unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias, eps: float) -> torch.Tensor:
    return F.layer_norm(x.float(), (x.shape[-1],), weight.float(), None if bias is None else bias.float(),
                        eps).to(x.dtype)


def activation(x: torch.Tensor, kind: str, gated: bool = False, alpha: float = 1.702, limit: float = 7.0):
    """kind: gelu | gelu_tanh | quick_gelu | silu | swiglu_oai.  gated: x = [gate | up]."""
    if gated:
        d = x.shape[-1] // 2
        g, u = x[..., :d].float(), x[..., d:].float()
    else:
        g, u = x.float(), None
    if kind == "swiglu_oai":
        g = g.clamp(max=limit)
        u = u.clamp(min=-limit, max=limit)
        return (g * torch.sigmoid(alpha * g) * (u + 1)).to(x.dtype)
    if kind == "gelu":
        y = F.gelu(g)
    elif kind == "gelu_tanh":
        y = F.gelu(g, approximate="tanh")
    elif kind == "quick_gelu":
        y = g * torch.sigmoid(1.702 * g)
    elif kind == "silu":
        y = F.silu(g)
    else:
        raise ValueError(f"unknown activation {kind!r}")
    return (y * u if u is not None else y).to(x.dtype)


def rms_norm_gated(x: torch.Tensor, z: torch.Tensor, w: torch.Tensor, eps: float, group: int = 0,
                   norm_before_gate: bool = True) -> torch.Tensor:
    """rmsnorm(x) * w * silu(z) (or rmsnorm(x * silu(z)) * w), optionally per group of columns."""
    H = x.shape[-1]
    g = group or H
    xf, zf = x.float().reshape(-1, g), z.float().reshape(-1, g)
    gate = F.silu(zf)
    if not norm_before_gate:
        xf = xf * gate
    y = xf * torch.rsqrt((xf * xf).mean(-1, keepdim=True) + eps) * w.float()[:g]
    if norm_before_gate:
        y = y * gate
    return y.reshape(x.shape).to(x.dtype)


# ---------------------------------------------------------------- beam search
def beam_select(logits: torch.Tensor, scores: torch.Tensor, k: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """logits [groups * beams, vocab], scores [groups, beams] -> the k best totals of each group (of the scores' type), their beams and tokens."""
    (groups, width), vocab = scores.shape, logits.shape[1]
    x = logits.double()
    x = x - torch.logsumexp(x, -1, keepdim=True)                # NaN where a row has no distribution
    total = torch.nan_to_num(scores.double().reshape(-1, 1) + x, nan=-torch.inf, posinf=-torch.inf, neginf=-torch.inf)
    best, at = torch.sort(total.reshape(groups, width * vocab), dim=-1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k]
    return best.to(scores.dtype), (at // vocab).to(torch.int32), at % vocab


def reorder_beams(tensors, rows: torch.Tensor, parents: torch.Tensor, lengths: Optional[torch.Tensor] = None, int4_dim: int = 0) -> None:
    """Rows (or the first ``lengths`` tokens of pages) of every tensor, in place; rows and parents out of range raise."""
    source, dest, tokens = [], [], []
    for g, (mine, follows) in enumerate(zip(rows.tolist(), parents.tolist())):
        for w, p in enumerate(follows):
            if not -1 <= p < len(mine) or mine[w] < -1 or p >= 0 and mine[w] >= 0 and mine[p] < 0:
                raise IndexError(f"group {g}: beam {w} in row {mine[w]} follows beam {p} of {len(mine)}")
            if p >= 0 and mine[w] >= 0 and p != w:
                source.append(mine[p])
                dest.append(mine[w])
                tokens.append(-1 if lengths is None else max(0, int(lengths[g])))
    for t in tensors:
        if any(r >= t.shape[0] for r in source + dest):
            raise IndexError(f"a row above {t.shape[0]}")
        old = t[torch.tensor(source, dtype=torch.int64)] if source else None
        for i, (r, n) in enumerate(zip(dest, tokens)):
            if n < 0:
                t[r] = old[i]
            elif t.dtype == torch.uint8:
                n = (n + KV_INT4_TOKENS - 1) // KV_INT4_TOKENS * 9 * int4_dim
                t[r, :, :n] = old[i, :, :n]
            else:
                t[r, :n] = old[i, :n]


def paged_attention_shared(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, query_start_loc, seq_lens, block_table: torch.Tensor,
                           group_starts, prefix_lens, scale: float, out: torch.Tensor) -> torch.Tensor:
    """Causal attention where the first ``prefix_lens[g]`` keys of the sequences of group g are read through its first sequence's pages."""
    cu, lens = [int(x) for x in query_start_loc], [int(x) for x in seq_lens]
    n, bs = len(lens), k_cache.shape[1]
    if any(not 0 <= a <= b <= n for a, b in zip(group_starts, group_starts[1:])):
        raise IndexError(f"group starts {group_starts} of {n} sequences")
    first, prefix = list(range(n)), [0] * n
    for a, b, p in zip(group_starts, group_starts[1:], prefix_lens):
        p = max(0, min([p] + [max(0, lens[s] - (cu[s + 1] - cu[s])) for s in range(a, b) if cu[s + 1] > cu[s]]))
        for s in range(a, b):
            first[s], prefix[s] = a, p
    G = q.shape[1] // k_cache.shape[2]
    for s in range(n):
        new = cu[s + 1] - cu[s]
        if new <= 0:
            continue
        pos = torch.arange(max(lens[s], 0), device=q.device)
        page = torch.where(pos < prefix[s], block_table[first[s]][pos // bs], block_table[s][pos // bs]).long()
        k, v = (t[page, pos % bs].float().repeat_interleave(G, 1) for t in (k_cache, v_cache))
        score = torch.einsum("qhd,khd->hqk", q[cu[s]:cu[s + 1]].float(), k) * scale
        hidden = pos[None] > torch.arange(lens[s] - new, lens[s], device=q.device)[:, None]
        score = score.masked_fill(hidden, -torch.inf)
        p = torch.where(hidden.all(-1)[None, :, None], 0.0, torch.softmax(score, -1))
        out[cu[s]:cu[s + 1]] = torch.einsum("hqk,khd->qhd", p, v).to(out.dtype)
    return out
