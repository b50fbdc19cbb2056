// Attention of prompts over a 4-bit paged cache (format: kv_int4.cuh), on tcgen05.
//
// Two query tiles of 128 rows (row = token * G + head of the group) share every tile of 128 keys, a warpgroup each, as in the kernel over
// bf16 pages (attention_prefill.cu, which has the reasons for that split).  Keys and values come packed by bulk copies, a quarter of
// the bytes, and a third warpgroup unpacks them into the swizzled tiles that the tensor cores read:
//   warps 0..3, 4..7   queries, softmax and epilogue of query tile 0, 1 (one thread per row)
//   warps 8..11        keys and values out of the packed ring into their tiles
//   warp 12            packed tiles into the ring;  warp 13  MMA issuer
// Unpacking 128 keys and values costs the four warps some 480 instructions each, next to the 128 exponentials a thread that bound the
// softmax warps; without it those pages would cost a pass of their own that writes and reads four times the bytes.
// Channels of keys lie as unpacking yields them (j and j + 4 of eight side by side), and so do the queries'.  With few
// tiles a sequence's keys are split into parts, which join in a second kernel.
// A value whose scale is no number would reach rows that do not see it (0 x NaN): near a mask's edges such groups enter as
// zeros, are noted, and put into the rows that see them at the end.
// All waits are bounded.
// Measured, 32 heads on 8 of 128: 8 prompts of 1000 tokens 135 us (bf16 pages: 127), one of 4096 tokens 153 us (149), 0.90 PFLOP/s; 137 tokens
// 11.3 us (those go to the kernel for few rows: 7.7).  28 heads on 4 of 64, three portions of 667 tokens behind 9000, window 4096: 143 us,
// where the exponentials alone take 52 us of the multifunction units.  Scores in halves of 64 keep a row in registers without spills: 128
// at once with the registers moved to the softmax warps (setmaxnreg) took 150 us there.  A block that works through several items (the
// next one's tiles unpacked while the last one's results are written) gained nothing: 143 us, or 198 with every 148th item fixed.
#include "attention_int4.cuh"

namespace b200 {

constexpr int P4_THREADS = 448;
constexpr int P4_HALF = 128 * 128;          // 128 rows x 64 bf16
constexpr int P4_RING = 3;                  // packed tiles
constexpr int P4_EDGE = 3;                  // tiles at either end that a pair of query tiles (256 tokens at most) may see in part

template <int D>
struct Int4PrefillCfg {
  static constexpr int NK = D / 64;
  static constexpr int TILE = NK * P4_HALF;
  static constexpr int UNIT = kv4_unit_bytes(D);
  static constexpr int PACKED = 8 * UNIT;
  static constexpr int NOTES = 2 * P4_EDGE * 128;
  static constexpr int SMEM_BYTES = 6 * TILE + P4_RING * PACKED + NOTES + 1024 + 512;
};

template <int D>
__global__ void __launch_bounds__(P4_THREADS, 1) attn_int4_prefill_kernel(const Int4Params p) {
  using Cfg = Int4PrefillCfg<D>;
  constexpr int NK = Cfg::NK, TILE = Cfg::TILE, UNIT = Cfg::UNIT, O_COL = 256;

  extern __shared__ uint8_t smem_raw[];
  __shared__ int item[4];                     // sequence, its first query row, query rows, keys
  const int warp = warp_index(), lane = threadIdx.x & 31;
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);      // still known to be shared memory
  uint8_t* Qs = smem;
  uint8_t* Ks = Qs + 2 * TILE;
  uint8_t* Vs = Ks + 2 * TILE;
  uint8_t* Ps = Vs + 2 * TILE;
  uint32_t* notes = (uint32_t*)(Ps + P4_RING * Cfg::PACKED);       // [slot][key] bytes of groups
  uint64_t* bars = (uint64_t*)(notes + Cfg::NOTES / 4);
  uint64_t* q_full = bars;             // 1
  uint64_t* k_full = bars + 1;         // 2
  uint64_t* k_empty = bars + 3;        // 2
  uint64_t* v_full = bars + 5;         // 2
  uint64_t* v_empty = bars + 7;        // 2
  uint64_t* s_full = bars + 9;         // 2: scores of query tile w
  uint64_t* p_full = bars + 11;        // 2: probabilities of query tile w
  uint64_t* o_full = bars + 13;        // 2: last product of query tile w
  uint64_t* pk_full = bars + 15;       // P4_RING
  uint64_t* pk_empty = bars + 18;      // P4_RING
  uint32_t* tmem_ptr = (uint32_t*)(bars + 21);
  volatile int* abort_word = (volatile int*)(tmem_ptr + 1);
  volatile int* noted = (volatile int*)(tmem_ptr + 2);

  // ---------------- work item: a pair of query tiles and a part of their keys; late pairs see more keys and come first.  Pairs of
  // sequence i begin at (cu[i] - base) / pair + i; the thread whose sequence has this one says so
  const int h = blockIdx.x, G = p.G, tpt = 128 / G, part = blockIdx.z;
  const int wi = gridDim.y - 1 - blockIdx.y, pair = 2 * tpt, base = p.cu[0];
  for (int i = threadIdx.x; i < p.num_seqs; i += P4_THREADS) {
    const int from = p.cu[i], to = p.cu[i + 1], keys = p.seq_lens[i];
    if ((from - base) / pair + i <= wi && (i + 1 == p.num_seqs || (to - base) / pair + i + 1 > wi)) {
      item[0] = i;
      item[1] = from;
      item[2] = to - from;
      item[3] = keys;
    }
  }
  if (threadIdx.x == 0) {
    mbar_init(q_full, 8);
    for (int b = 0; b < 2; b++) {
      mbar_init(&k_full[b], 4);
      mbar_init(&k_empty[b], 1);
      mbar_init(&v_full[b], 4);
      mbar_init(&v_empty[b], 1);
      mbar_init(&s_full[b], 1);
      mbar_init(&p_full[b], 4);
      mbar_init(&o_full[b], 1);
    }
    for (int b = 0; b < P4_RING; b++) {
      mbar_init(&pk_full[b], 1);
      mbar_init(&pk_empty[b], 4);
    }
    *abort_word = 0;
    *noted = 0;
    mbar_fence_init();
  }
  for (int i = threadIdx.x; i < Cfg::NOTES / 4; i += P4_THREADS) notes[i] = 0;
  if (warp == 13) {
    tmem_alloc(tmem_ptr, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = warp_uniform(*tmem_ptr);
  const int seq = item[0], q_start = item[1], q_len = item[2], seq_len = item[3], ctx = seq_len - q_len;
  const int tok0 = (wi - ((q_start - base) / pair + seq)) * pair;
  const bool beyond = q_start < 0 || q_start + (long)q_len > p.q_rows;          // reported; nothing lies there
  if (tok0 >= q_len || beyond) {              // the grid has a pair more than some sequences
    if (beyond && threadIdx.x == 0 && p.status) atomicExch(p.status, B200_BAD_INDEX);
    if (warp == 13) tmem_dealloc(tmem_base, 512);
    return;
  }
  int ntok[2], t_end[2];
#pragma unroll
  for (int w = 0; w < 2; w++) {
    ntok[w] = max(0, min(tpt, q_len - tok0 - w * tpt));
    const int end = p.causal ? min(seq_len, ctx + tok0 + w * tpt + ntok[w]) : seq_len;
    t_end[w] = ntok[w] > 0 ? max(0, end + 127) >> 7 : 0;
  }
  const int key_lo = p.window > 0 ? max(0, ctx + tok0 - p.window + 1) : 0;                     // keys that any row sees
  const int key_hi = p.causal ? min(seq_len, ctx + tok0 + ntok[0] + ntok[1]) : seq_len;
  const int t_lo = key_lo >> 7, all = max(0, max(t_end[0], t_end[1]) - t_lo);
  const int t_a = t_lo + (int)((long)all * part / p.parts), t_b = t_lo + (int)((long)all * (part + 1) / p.parts);
  const int n = t_b - t_a;
  const int n0 = max(0, min(t_b, t_end[0]) - t_a), n1 = max(0, min(t_b, t_end[1]) - t_a);      // key tiles of each query tile
  auto note_slot = [&](int tile) {            // where a tile's values that are no numbers are noted; -1: nowhere
    const int i = tile - t_lo;
    return i < P4_EDGE ? i : i >= all - P4_EDGE ? i - (all - 2 * P4_EDGE) : -1;
  };

  if (warp >= 12) {
    if (warp == 12) {
      // ---------------------------------------------------------- packed tiles
      const int upp = p.block_size / KV4_TOKENS;
      const int* bt = p.block_table + seq * p.table_stride;
      const bool whole = upp % 8 == 0;           // a tile lies in one page
      for (int j = 0; j < n; j++) {
        const int u0 = (t_a + j) * 8, units = min(8, (key_hi + KV4_TOKENS - 1) / KV4_TOKENS - u0);
        const int mine = whole ? u0 : u0 + lane, col = mine / upp;
        int blk = 0;
        if (whole || lane < units) blk = col < p.max_blocks ? bt[col] : -1;
        const bool bad = __any_sync(0xffffffffu, blk < 0 || blk >= p.num_blocks);
        const long from = (((long)blk * p.Hkv + h) * upp + (mine - col * upp)) * UNIT;
        for (int kv = 0; kv < 2; kv++) {
          const int i = 2 * j + kv, slot = i % P4_RING;
          if (!__all_sync(0xffffffffu, mbar_wait(&pk_empty[slot], ((uint32_t)(i / P4_RING) & 1u) ^ 1u, abort_word))) goto done;
          if (bad) {
            *abort_word = B200_BAD_INDEX;
            goto done;
          }
          uint8_t* dst = Ps + slot * Cfg::PACKED;
          const uint8_t* src = (kv ? p.v_cache : p.k_cache) + from;
          if (lane == 0) mbar_expect_tx(&pk_full[slot], units * UNIT);
          __syncwarp();
          if (whole) {
            if (lane == 0) i4_bulk_load(dst, src, units * UNIT, &pk_full[slot]);
          } else if (lane < units) {
            i4_bulk_load(dst + lane * UNIT, src, UNIT, &pk_full[slot]);
          }
          __syncwarp();
        }
      }
    } else if (warp == 13 && n > 0) {
      // ---------------------------------------------------------- MMA issuer: one thread walks the loop (see warp_uniform)
      if (elect_one()) {
        constexpr uint32_t idesc_s = make_idesc_f16(128, 128, true, false, false);
        constexpr uint32_t idesc_o = make_idesc_f16(128, D, true, false, true);
        const uint64_t dq0 = make_smem_desc(smem_u32(Qs), 16, 1024, kLayoutSw128), dk0 = make_smem_desc(smem_u32(Ks), 16, 1024, kLayoutSw128);
        const uint64_t dv0 = make_smem_desc(smem_u32(Vs), P4_HALF, 1024, kLayoutSw128);
        auto issue_s = [&](int w, int j) {
          const uint64_t dq = dq0 + (uint32_t)(w * (TILE >> 4)), dk = dk0 + (uint32_t)((j & 1) * (TILE >> 4));
#pragma unroll
          for (int kk = 0; kk < NK * 4; kk++) {
            const uint32_t o = ((kk >> 2) * P4_HALF + (kk & 3) * 32) >> 4;
            umma_f16_ss(tmem_base + w * 128, dq + o, dk + o, idesc_s, kk > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[w]);
        };
        if (!mbar_wait(q_full, 0, abort_word)) goto done;
        if (!mbar_wait(&k_full[0], 0, abort_word)) goto done;
        tc_fence_after();
        if (n0 > 0) issue_s(0, 0);
        if (n1 > 0) issue_s(1, 0);
        umma_commit(&k_empty[0]);
        for (int j = 0; j < n; j++) {
          const int vs = j & 1;
          if (!mbar_wait(&v_full[vs], (uint32_t)(j >> 1) & 1u, abort_word)) goto done;
          if (j + 1 < n && !mbar_wait(&k_full[(j + 1) & 1], (uint32_t)((j + 1) >> 1) & 1u, abort_word)) goto done;
          const uint64_t dv = dv0 + (uint32_t)(vs * (TILE >> 4));
#pragma unroll 1
          for (int w = 0; w < 2; w++) {
            const int nw = w == 0 ? n0 : n1;
            if (j < nw) {
              if (!mbar_wait(&p_full[w], (uint32_t)j & 1u, abort_word)) goto done;
              tc_fence_after();
#pragma unroll
              for (int kk = 0; kk < 8; kk++)
                umma_f16_ts(tmem_base + O_COL + w * 128, tmem_base + w * 128 + (kk & 3) * 8 + (kk >> 2) * 64, dv + kk * 128, idesc_o, (j > 0 || kk > 0) ? 1u : 0u);
              if (j == nw - 1) umma_commit(&o_full[w]);
              if (j + 1 < nw) issue_s(w, j + 1);
            }
          }
          umma_commit(&v_empty[vs]);
          if (j + 1 < n) umma_commit(&k_empty[(j + 1) & 1]);
        }
      }
    }
  } else if (warp >= 8) {
    // ------------------------------------------------------------ unpacking
    if (n > 0) {
      const int wl = warp - 8;
      for (int j = 0; j < n; j++) {
        const int st = j & 1, slot_n = note_slot(t_a + j);
#pragma unroll 1
        for (int kv = 0; kv < 2; kv++) {
          const int i = 2 * j + kv, slot = i % P4_RING;
          if (!__all_sync(0xffffffffu, mbar_wait(&pk_full[slot], (uint32_t)(i / P4_RING) & 1u, abort_word))) goto done;
          if (!__all_sync(0xffffffffu, mbar_wait(kv ? &v_empty[st] : &k_empty[st], ((uint32_t)(j >> 1) & 1u) ^ 1u, abort_word))) goto done;
          const uint8_t* src = Ps + slot * Cfg::PACKED;
          if (kv == 0) {
            // keys: a lane takes 16 packed bytes (32 channels) of a row; at D = 128 the lanes of the second slab write their chunks in
            // another order, so that eight lanes meet eight chunks' banks
            constexpr int Q = D / 32, RP = 32 / Q;          // lanes of a row, rows of a warp's pass
            const int q = lane % Q;
            uint8_t* dst = Ks + st * TILE + (q >> 1) * P4_HALF;
#pragma unroll 2
            for (int pass = 0; pass < 128 / (4 * RP); pass++) {
              const int row = (pass * 4 + wl) * RP + lane / Q, t = row & 15;
              const uint8_t* unit = src + (row >> 4) * UNIT;
              const uint4 x = *reinterpret_cast<const uint4*>(unit + kv4_key_word(D, t, q * 32));
              const Kv4Scale s(*reinterpret_cast<const uint16_t*>(unit + kv4_scale(D, t, q)) * 0x10001u);
              const bool late = q >= 2;
              const uint32_t w4[4] = {late ? x.z : x.x, late ? x.w : x.y, late ? x.x : x.z, late ? x.y : x.w};
#pragma unroll
              for (int c = 0; c < 4; c++) {
                const uint32_t hi = w4[c] >> 8;
                const uint4 y = make_uint4(kv4_pair(0, w4[c], s), kv4_pair(1, w4[c], s), kv4_pair(0, hi, s), kv4_pair(1, hi, s));
                const int chunk = (q & 1) * 4 + (late ? c ^ 2 : c);
                *reinterpret_cast<uint4*>(dst + row * 128 + ((chunk ^ (row & 7)) << 4)) = y;
              }
            }
          } else {
            // values: a lane takes 16 channels of two tokens
            constexpr int Q = D / 16, RP = 32 / Q;          // lanes of a pair, pairs of a warp's pass
            const int q = lane % Q;
            uint8_t* dst = Vs + st * TILE + (q >> 2) * P4_HALF;
#pragma unroll 2
            for (int pass = 0; pass < 64 / (4 * RP); pass++) {
              const int pr = (pass * 4 + wl) * RP + lane / Q, t = 2 * (pr & 7), row = 2 * pr, key = (t_a + j) * 128 + row;
              const uint8_t* unit = src + (row >> 4) * UNIT;
              const uint4 x = *reinterpret_cast<const uint4*>(unit + kv4_value_word(D, t, q * 16));
              uint32_t sw = *reinterpret_cast<const uint32_t*>(unit + kv4_scale(D, t, q >> 1));
              if (slot_n >= 0) {                 // tokens that no row sees weigh nothing, whatever lies in their place
                if (key < key_lo || key >= key_hi) sw &= 0xffff0000u;
                if (key + 1 < key_lo || key + 1 >= key_hi) sw &= 0x0000ffffu;
                const bool odd0 = (sw & 0x7f80u) == 0x7f80u, odd1 = (sw & 0x7f800000u) == 0x7f800000u;
                if (odd0 || odd1) {
                  if (odd0) sw &= 0xffff0000u;
                  if (odd1) sw &= 0x0000ffffu;
                  atomicOr(&notes[slot_n * 32 + (row >> 2)], ((odd0 ? 1u : 0u) | (odd1 ? 256u : 0u)) << ((q >> 1) + 8 * (row & 2)));
                  *noted = 1;
                }
              }
              const Kv4Scale s(sw);
              const bool late = D == 128 ? q >= 4 : (pr & 1) != 0;        // which of the two chunks first: banks again
              const uint32_t w4[4] = {late ? x.z : x.x, late ? x.w : x.y, late ? x.x : x.z, late ? x.y : x.w};
#pragma unroll
              for (int c = 0; c < 2; c++) {
                uint32_t e[4], o[4];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                  const uint32_t lw = w4[2 * c + k], hw = lw >> 8;
                  const uint32_t p0 = kv4_pair(0, lw, s), p1 = kv4_pair(1, lw, s), p2 = kv4_pair(0, hw, s), p3 = kv4_pair(1, hw, s);
                  e[2 * k] = __byte_perm(p0, p1, 0x5410);
                  o[2 * k] = __byte_perm(p0, p1, 0x7632);
                  e[2 * k + 1] = __byte_perm(p2, p3, 0x5410);
                  o[2 * k + 1] = __byte_perm(p2, p3, 0x7632);
                }
                const int chunk = (q & 3) * 2 + (late ? c ^ 1 : c);
                *reinterpret_cast<uint4*>(dst + row * 128 + ((chunk ^ (row & 7)) << 4)) = make_uint4(e[0], e[1], e[2], e[3]);
                *reinterpret_cast<uint4*>(dst + (row + 1) * 128 + ((chunk ^ ((row + 1) & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
              }
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(kv ? &v_full[st] : &k_full[st]);
            mbar_arrive(&pk_empty[slot]);
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------ softmax / epilogue of query tile w
    const int w = warp >> 2;
    const int nw = w == 0 ? n0 : n1, nt = w == 0 ? ntok[0] : ntok[1];
    {
      // its queries, channels j and j + 4 side by side; eight lanes take a slab's row
      uint8_t* dst = Qs + w * TILE;
      const int c8 = lane & 7;
#pragma unroll
      for (int s = 0; s < NK; s++) {
        uint4 x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int rr = (warp & 3) * 32 + i * 4 + (lane >> 3), tok = rr / G, g = rr - tok * G;
          x[i] = make_uint4(0, 0, 0, 0);
          if (tok < nt)
            x[i] = *reinterpret_cast<const uint4*>(p.q + (long)(q_start + tok0 + w * tpt + tok) * p.q_stride + (long)(h * G + g) * D + s * 64 + c8 * 8);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int rr = (warp & 3) * 32 + i * 4 + (lane >> 3);
          uint4 y;
          y.x = __byte_perm(x[i].x, x[i].z, 0x5410);
          y.y = __byte_perm(x[i].x, x[i].z, 0x7632);
          y.z = __byte_perm(x[i].y, x[i].w, 0x5410);
          y.w = __byte_perm(x[i].y, x[i].w, 0x7632);
          *reinterpret_cast<uint4*>(dst + s * P4_HALF + rr * 128 + ((c8 ^ (rr & 7)) << 4)) = y;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    if (nt > 0) {
      const int row = (warp & 3) * 32 + lane;
      const int tok = row / G, g = row - tok * G;
      const int t_first = tok0 + w * tpt;
      const bool row_valid = tok < nt;
      const int q_pos = ctx + t_first + tok;
      const uint32_t t_lane = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
      const uint32_t t_s = t_lane + w * 128, t_o = t_lane + O_COL + w * 128;
      const float sl2 = p.scale_log2;
      int k_hi = seq_len;                      // keys [k_lo, k_hi) are visible to this row
      if (p.causal) k_hi = min(k_hi, q_pos + 1);
      const int k_lo = p.window > 0 ? max(0, q_pos - p.window + 1) : 0;
      // seen by every row of the warp that there is
      const int tok_a = (warp & 3) * 32 / G, tok_b = min(nt - 1, ((warp & 3) * 32 + 31) / G);
      const int all_hi = p.causal ? min(seq_len, ctx + t_first + tok_a + 1) : seq_len;
      const int all_lo = p.window > 0 ? max(0, ctx + t_first + tok_b - p.window + 1) : 0;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < nw; j++) {
        if (!__all_sync(0xffffffffu, mbar_wait(&s_full[w], (uint32_t)j & 1u, abort_word))) goto done;
        tc_fence_after();
        // 64 scores at a time: the maximum of all, then the second half's probabilities out of the registers that still hold it, then the
        // first half's.  A half's probabilities replace its own scores (keys 64 on: column 64 on), two to a column
        const int key0 = (t_a + j) << 7;
        uint32_t sr[64];
        auto half = [&](int hf) {
          tmem_ld_32x32b_x32(t_s + 64 * hf, sr);
          tmem_ld_32x32b_x32(t_s + 64 * hf + 32, sr + 32);
          tmem_ld_wait();
          const int first = key0 + 64 * hf;
          if (first + 64 > all_hi || first < all_lo) {
            const int end = k_hi - first, start = k_lo - first;
#pragma unroll
            for (int c = 0; c < 2; c++) {        // 32 keys at a time, where some row of the warp does not see them all
              if (first + 32 * c + 32 > all_hi) {
#pragma unroll
                for (int i = 32 * c; i < 32 * c + 32; i++) if (i >= end) sr[i] = 0xff800000u;   // -inf
              }
              if (first + 32 * c < all_lo) {
#pragma unroll
                for (int i = 32 * c; i < 32 * c + 32; i++) if (i < start) sr[i] = 0xff800000u;
              }
            }
          }
        };
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
          half(hf);
#pragma unroll
          for (int i = 0; i < 64; i += 8)
#pragma unroll
            for (int q = 0; q < 4; q++)
              mx[q] = fmaxf(mx[q], fmaxf(__uint_as_float(sr[i + 2 * q]), __uint_as_float(sr[i + 2 * q + 1])));
        }
        const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        // O is rescaled only where a score outgrew the maximum by more than a factor of 2^8: no probability then overflows bf16
        float alpha = 1.f;
        bool need = false;
        if (mt > m && (m == -INFINITY || (mt - m) * sl2 > 8.f)) {
          alpha = m == -INFINITY ? 0.f : i4_exp2((m - mt) * sl2);
          need = m != -INFINITY;               // an all-masked row has accumulated zeros only
          m = mt;
        }
        l *= alpha;
        if (j > 0 && __any_sync(0xffffffffu, need && row_valid)) {
          const float a = need ? alpha : 1.f;
#pragma unroll 1
          for (int c = 0; c < D / 32; c++) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(t_o + c * 32, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; i++) r[i] = __float_as_uint(__uint_as_float(r[i]) * a);
            tmem_st_32x32b_x32(t_o + c * 32, r);
          }
          // the second half once more, rather than in registers across this rare case: 4096 tokens 162 -> 153 us (D = 64: 142 -> 146)
          if constexpr (D == 128) half(1);
        }
        const float nmb = m == -INFINITY ? 0.f : -m * sl2;
        float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int hf = 1; hf >= 0; hf--) {
          if (hf == 0) half(0);
#pragma unroll
          for (int c = 0; c < 2; c++) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
              const float p0 = i4_exp2(fmaf(__uint_as_float(sr[c * 32 + 2 * i]), sl2, nmb));
              const float p1 = i4_exp2(fmaf(__uint_as_float(sr[c * 32 + 2 * i + 1]), sl2, nmb));
              rs[(i & 1) * 2] += p0;
              rs[(i & 1) * 2 + 1] += p1;
              pk[i] = pack_bf16x2(p0, p1);
            }
            tmem_st_32x32b_x16(t_s + 64 * hf + c * 16, pk);
          }
        }
        l += (rs[0] + rs[1]) + (rs[2] + rs[3]);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[w]);
      }
      if (nw > 0) {
        if (!__all_sync(0xffffffffu, mbar_wait(&o_full[w], 0, abort_word))) goto done;
        tc_fence_after();
      }
      uint32_t poison = 0;                     // groups with a value that is no number among the keys that this row sees
      if (nw > 0 && *noted != 0) {
        for (int j = 0; j < nw; j++) {
          const int slot = note_slot(t_a + j);
          if (slot < 0) continue;
          const int key0 = (t_a + j) << 7, i0 = max(0, k_lo - key0), i1 = min(128, k_hi - key0);
          for (int i = i0; i < i1; i++) poison |= notes[slot * 32 + (i >> 2)] >> (8 * (i & 3)) & 0xffu;
        }
      }
      const float inv = l == 0.f ? 0.f : KV4_UNDO / l;       // a row without keys: zeros
      const long head = (long)(h * G + g), token = q_start + t_first + tok;
      const long at = (token * (p.Hkv * G) + head) * p.parts + part;
      if (p.parts > 1 && row_valid) p.part_lse[at] = l == 0.f ? -INFINITY : fmaf(m, sl2, log2f(l));
#pragma unroll 1
      for (int c = 0; c < D / 32; c++) {
        uint32_t r[32];
        if (nw > 0) {
          tmem_ld_32x32b_x32(t_o + c * 32, r);
          tmem_ld_wait();
        }
        float f[32];
#pragma unroll
        for (int i = 0; i < 32; i++) f[i] = nw > 0 ? __uint_as_float(r[i]) * inv : 0.f;
        if (poison >> c & 1u) {
#pragma unroll
          for (int i = 0; i < 32; i++) f[i] = __int_as_float(0x7fc00000);
        }
        if (row_valid) {
          if (p.parts == 1) {
            __nv_bfloat16* dst = p.out + token * p.out_stride + head * D + c * 32;
#pragma unroll
            for (int q4 = 0; q4 < 4; q4++) {
              uint4 o;
              o.x = pack_bf16x2(f[q4 * 8 + 0], f[q4 * 8 + 1]);
              o.y = pack_bf16x2(f[q4 * 8 + 2], f[q4 * 8 + 3]);
              o.z = pack_bf16x2(f[q4 * 8 + 4], f[q4 * 8 + 5]);
              o.w = pack_bf16x2(f[q4 * 8 + 6], f[q4 * 8 + 7]);
              *reinterpret_cast<uint4*>(dst + q4 * 8) = o;
            }
          } else if (l != 0.f) {
            float4* dst = reinterpret_cast<float4*>(p.part_o + at * D + c * 32);
#pragma unroll
            for (int q4 = 0; q4 < 8; q4++) dst[q4] = make_float4(f[q4 * 4], f[q4 * 4 + 1], f[q4 * 4 + 2], f[q4 * 4 + 3]);
          }
        }
      }
    }
  }
done:
  __syncwarp();             // the elected threads come back to their warps
  tc_fence_before();
  __syncthreads();
  if (*abort_word != 0) {
    // let copies still in flight land before the block's shared memory is released
    const uint64_t t_start = globaltimer_ns();
    while (globaltimer_ns() - t_start < 50000ull) __nanosleep(1000);
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, *abort_word);
    __syncthreads();
  }
  if (warp == 13) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int D>
static int launch_int4_prefill(const Int4Params& p, long tokens, cudaStream_t stream) {
  using Cfg = Int4PrefillCfg<D>;
  cudaError_t e = allow_smem<attn_int4_prefill_kernel<D>>(Cfg::SMEM_BYTES);
  if (e != cudaSuccess) return (int)e;
  const long pairs = tokens / (2 * (128 / p.G)) + p.num_seqs;
  if (pairs > 65535) return 9887;
  attn_int4_prefill_kernel<D><<<dim3((unsigned)p.Hkv, (unsigned)pairs, (unsigned)p.parts), P4_THREADS, Cfg::SMEM_BYTES, stream>>>(p);
  return B200_CHECK_LAUNCH();
}

}  // namespace b200

using namespace b200;

// The same for prompts: tokens bounds cu[num_seqs] - cu[0]; groups of up to 128 heads.
B200_API int b200_attn_int4_prefill(const Int4Args* a) {
  if (a->num_seqs <= 0 || a->q_rows <= 0 || a->tokens <= 0) return 0;
  Int4Params p;
  int rc = int4_params(&p, *a);
  if (rc) return rc;
  if (p.G > 128) return 9883;
  if (p.parts > 1 && !a->scratch) return 9885;
  rc = a->D == 128 ? launch_int4_prefill<128>(p, a->tokens, a->stream) : launch_int4_prefill<64>(p, a->tokens, a->stream);
  return rc || p.parts == 1 ? rc : int4_join(p, a->D, a->q_rows, a->stream);
}
