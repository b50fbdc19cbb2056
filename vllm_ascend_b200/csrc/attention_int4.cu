// Attention of few query rows over a 4-bit paged cache (format: kv_int4.cuh): decode, drafts to verify, any batch whose
// sequences have few new tokens.
//
//   o_r = sum_j p_rj v_j / sum_j p_rj,   p_rj = exp(scale q_r k_j - m_r),   m_r the running maximum
//
// Bound: memory, 9/8 D bytes a stored token and head, and close behind it the instructions that unpack (three for two channels).
// So nothing is unpacked to shared memory: a warp unpacks into the very registers that the tensor cores read, and both products have
// the stored side as the rows of A, which takes 16 of them for 8 query rows:
//   S^T = K Q^T     16 tokens x 8 rows, over D.  A lane holds 32 (D = 64: 16) adjacent channels of two tokens; the order of the
//                   sum is free, so the query fragments follow what unpacking yields (channels j and j + 4 of eight)
//   O^T = V^T P^T   D channels x 8 rows, over tokens.  A lane holds 16 (8) adjacent channels of four tokens; S^T's results
//                   become P^T's fragments by transposing 8 x 8 blocks between the lanes
// A block is one (sequence, KV head, part of the sequence); each of its warps walks a stretch of it, in tiles of 64 tokens where
// all rows see them and 16 at a time at the edges, through a ring of its own that bulk copies fill, with a running maximum of
// its own; they join at the end.  Up to sixteen parts are a cluster whose blocks join through each other's shared memory; more (few very
// long sequences) join in a second kernel.
// Measured: 256 sequences of 1152 tokens, 32 heads on 8 of 128: 76 us, 4.4 TB/s (the copies alone, nothing unpacked: 6.5; unpacking and
// products alone: 46 us; twelve warps of an SM overlap the two that far, and 16 with fewer registers no further; the last blocks of
// unequal sequences take some 10 of the 76); bf16 pages take 187 us.  3 of 60001 tokens, 64 heads: 57 us, 3.6 TB/s, 6 of it the second
// kernel (60 in a graph, in clusters).  One of 1337 tokens, 32 heads: 6.2 us.
#include "attention_int4.cuh"
#include "cluster_sum.cuh"

#include <type_traits>

namespace b200 {

constexpr int D4_WARPS = 4;

__device__ __forceinline__ void i4_mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t i4_transpose(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// NT tiles of 8 query rows: one with three blocks on an SM, two with two, whose warps have the registers for them (40 sequences of 2304
// tokens, 32 rows of 4 heads: 56 us with three blocks and tiles of 32 tokens, 49 us).  More rows are blocks of their own that read
// the pages again: four tiles (255 registers, spills, rows' fragments in shared memory) took 55 us there.
template <int D, int NT>
struct Int4Cfg {
  static constexpr int U = 4;                            // units of a tile
  static constexpr int BLOCKS = NT == 1 ? 3 : 2;         // of an SM
  static constexpr int UNIT = kv4_unit_bytes(D);
  static constexpr int STAGE = 2 * U * UNIT;             // keys, then values
  static constexpr int STAGES = 2 * (128 / D);
  static constexpr int RING = STAGES * STAGE;
  static constexpr int ROWS = 8 * NT;
  static constexpr int SMEM = D4_WARPS * RING + 1024;    // barriers, maxima and sums behind the rings
  static_assert(2 * ROWS * D * 4 <= RING, "a warp's result takes its ring's place, and the block's that behind the first warp's");
  static_assert(D4_WARPS * (STAGES * 8 + ROWS * 8) + ROWS * 8 + 16 <= 1024, "");
};

template <int D, int NT>
__global__ void __launch_bounds__(32 * D4_WARPS, Int4Cfg<D, NT>::BLOCKS) attn_int4_kernel(const Int4Params p) {
  using Cfg = Int4Cfg<D, NT>;
  constexpr int KW = D / 32;                    // groups: words of a token's keys in a lane
  constexpr int VX = D / 32;                    // words of two tokens' values in a lane
  constexpr int MT = D / 16;                    // channel tiles of the result
  constexpr int U = Cfg::U, ROWS = Cfg::ROWS;
  extern __shared__ __align__(128) uint8_t i4_smem[];
  const int warp = warp_index(), lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  uint8_t* ring = i4_smem + warp * Cfg::RING;
  uint64_t* bars = (uint64_t*)(i4_smem + D4_WARPS * Cfg::RING) + warp * Cfg::STAGES;
  float* ms = (float*)(i4_smem + D4_WARPS * (Cfg::RING + Cfg::STAGES * 8));        // [warps][rows], sums behind
  float* ls = ms + D4_WARPS * ROWS;
  float* block_m = ls + D4_WARPS * ROWS;                                           // [rows] of the block, sums behind
  float* block_l = block_m + ROWS;
  volatile int* abort_word = (volatile int*)(block_l + ROWS);
  volatile int* bad_page = abort_word + 1;       // apart from the word that ends waits: every warp still sees its own copies land

  const int seq = p.row_blocks == 1 ? blockIdx.x : blockIdx.x / p.row_blocks, row0 = (blockIdx.x - seq * p.row_blocks) * ROWS;
  const int h = blockIdx.y, part = blockIdx.z;
  const int q_start = p.cu[seq], q_len = p.cu[seq + 1] - q_start, len = p.seq_lens[seq], ctx = len - q_len;
  const int rows = min(q_len * p.G - row0, ROWS);
  if (rows <= 0) return;
  if (q_start < 0 || q_start + (long)q_len > p.q_rows) {         // reported; nothing lies there
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, B200_BAD_INDEX);
    return;
  }
  if (lane == 0)
    for (int s = 0; s < Cfg::STAGES; s++) mbar_init(&bars[s], 1);
  if (threadIdx.x == 0) *abort_word = *bad_page = 0;
  mbar_fence_init();
  __syncthreads();

  // keys that any row of the block sees, and those that all rows see
  const int tok_first = int4_div(row0, p.G, p.g_inv), tok_last = int4_div(row0 + rows - 1, p.G, p.g_inv);
  const int hi = max(0, p.causal ? min(len, ctx + tok_last + 1) : len), all_hi = p.causal ? min(len, ctx + tok_first + 1) : len;
  const int lo = p.window > 0 ? max(0, ctx + tok_first - p.window + 1) : 0, all_lo = p.window > 0 ? max(0, ctx + tok_last - p.window + 1) : 0;
  // the block's units, and the warp's among them
  const int u_lo = lo / KV4_TOKENS, units = max(0, (hi + KV4_TOKENS - 1) / KV4_TOKENS - u_lo);
  int b0 = 0, b1 = units;
  if (p.parts > 1) {
    b0 = (int)((uint32_t)units * part / (uint32_t)p.parts);
    b1 = (int)((uint32_t)units * (part + 1) / (uint32_t)p.parts);
  }
  const int first = u_lo + b0 + (b1 - b0) * warp / D4_WARPS, last = u_lo + b0 + (b1 - b0) * (warp + 1) / D4_WARPS;

  // the next tile to copy: lanes below U know the page of a unit each, and the unit's place there, walked by additions
  const int upp = p.block_size / KV4_TOKENS;
  const int* bt = p.block_table + seq * p.table_stride;
  int next = first, col = int4_div(first + lane, upp, p.upp_inv), at = first + lane - col * upp, blk = 0;
  const int step = int4_div(U, upp, p.upp_inv), rest = U - step * upp;
  auto look_up = [&]() {
    if (lane < U && next + lane < last) blk = col < p.max_blocks ? bt[col] : -1;
  };
  look_up();
  bool bad = false;
  auto issue = [&](int stage) {
    const int n = min(U, last - next);
    if (__any_sync(0xffffffffu, lane < n && (blk < 0 || blk >= p.num_blocks))) {
      bad = true;
      return;
    }
    const long from = (((long)blk * p.Hkv + h) * upp + at) * Cfg::UNIT;
    uint8_t* to = ring + stage * Cfg::STAGE;
    if (upp >= U) {                              // one run of a page, or two
      const int n0 = min(n, upp - __shfl_sync(0xffffffffu, at, 0));
      const long from0 = __shfl_sync(0xffffffffu, from, 0), from1 = __shfl_sync(0xffffffffu, from, n0 % U);
      if (elect_one()) {
        mbar_expect_tx(&bars[stage], 2 * n * Cfg::UNIT);
        i4_bulk_load(to, p.k_cache + from0, n0 * Cfg::UNIT, &bars[stage]);
        i4_bulk_load(to + U * Cfg::UNIT, p.v_cache + from0, n0 * Cfg::UNIT, &bars[stage]);
        if (n0 < n) {
          i4_bulk_load(to + n0 * Cfg::UNIT, p.k_cache + from1, (n - n0) * Cfg::UNIT, &bars[stage]);
          i4_bulk_load(to + (U + n0) * Cfg::UNIT, p.v_cache + from1, (n - n0) * Cfg::UNIT, &bars[stage]);
        }
      }
    } else {
      if (lane == 0) mbar_expect_tx(&bars[stage], 2 * n * Cfg::UNIT);
      __syncwarp();
      if (lane < n) {
        i4_bulk_load(to + lane * Cfg::UNIT, p.k_cache + from, Cfg::UNIT, &bars[stage]);
        i4_bulk_load(to + (U + lane) * Cfg::UNIT, p.v_cache + from, Cfg::UNIT, &bars[stage]);
      }
    }
    next += U;
    col += step;
    at += rest;
    if (at >= upp) {
      at -= upp;
      col++;
    }
    look_up();
  };
  for (int s = 0; s < Cfg::STAGES && next < last && !bad; s++) issue(s);

  // the rows' fragments: row r (+ 8 per tile), channels in the order of unpacking (j and j + 4 of a word's eight)
  uint32_t qf[NT][KW][4];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    const int row = row0 + nt * 8 + r, tok = int4_div(row, p.G, p.g_inv), g = row - tok * p.G;
    const bool here = nt * 8 + r < rows;
    const uint4* src = reinterpret_cast<const uint4*>(p.q + (long)(q_start + tok) * p.q_stride + (long)(h * p.G + g) * D + c * (D / 4));
#pragma unroll
    for (int w = 0; w < KW; w++) {
      const uint4 x = here ? src[w] : make_uint4(0, 0, 0, 0);
      qf[nt][w][0] = __byte_perm(x.x, x.z, 0x5410);
      qf[nt][w][1] = __byte_perm(x.x, x.z, 0x7632);
      qf[nt][w][2] = __byte_perm(x.y, x.w, 0x5410);
      qf[nt][w][3] = __byte_perm(x.y, x.w, 0x7632);
    }
  }
  // keys that columns 2 c and 2 c + 1 see
  int k_lo[NT][2], k_hi[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int i = nt * 8 + 2 * c + e, pos = ctx + int4_div(row0 + i, p.G, p.g_inv);
      k_hi[nt][e] = i < rows ? (p.causal ? min(len, pos + 1) : len) : 0;
      k_lo[nt][e] = p.window > 0 ? pos - p.window + 1 : 0;
    }

  float o[NT][MT][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    // rows that do not exist score 0, or -inf at an edge: a maximum of 0 never moves, so no row's rounding follows from how many
    // rows its block has room for
#pragma unroll
    for (int e = 0; e < 2; e++) m[nt][e] = nt * 8 + 2 * c + e < rows ? -INFINITY : 0.f;
    l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) o[nt][i][e] = 0.f;
  }
  const int kg = (c * (D / 4)) / KV4_GROUP, vg = (r * (D / 8)) / KV4_GROUP;

  // N units from ks and vs on, tokens from t0 on.  EDGE: some rows do not see all of them
  auto tokens = [&](auto n_units, auto edge, const uint8_t* ks, const uint8_t* vs, int t0) {
    constexpr int N = decltype(n_units)::value;
    constexpr bool EDGE = decltype(edge)::value;
    float s[N][NT][4];
#pragma unroll
    for (int u = 0; u < N; u++) {
      const uint8_t* unit = ks + u * Cfg::UNIT;
      uint32_t wa[KW], wb[KW];                   // words of tokens r and r + 8
      const uint8_t* ra = unit + kv4_key_word(D, r, c * (D / 4));
      if constexpr (KW == 4) {
        const uint4 a = *reinterpret_cast<const uint4*>(ra), b = *reinterpret_cast<const uint4*>(ra + 8 * (D / 2));
        wa[0] = a.x; wa[1] = a.y; wa[2] = a.z; wa[3] = a.w;
        wb[0] = b.x; wb[1] = b.y; wb[2] = b.z; wb[3] = b.w;
      } else {
        const uint2 a = *reinterpret_cast<const uint2*>(ra), b = *reinterpret_cast<const uint2*>(ra + 8 * (D / 2));
        wa[0] = a.x; wa[1] = a.y;
        wb[0] = b.x; wb[1] = b.y;
      }
      const uint16_t* sc = reinterpret_cast<const uint16_t*>(unit + kv4_scale(D, r, kg));
      const Kv4Scale sa(sc[0] * 0x10001u), sb(sc[8] * 0x10001u);
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[u][nt][e] = 0.f;
#pragma unroll
      for (int w = 0; w < KW; w++) {
#pragma unroll
        for (int j = 0; j < 2; j++) {            // channels 0, 1, 4, 5: the word's own low bytes; 2, 3, 6, 7
          const uint32_t xa = j ? wa[w] >> 8 : wa[w], xb = j ? wb[w] >> 8 : wb[w];
          const uint32_t a0 = kv4_pair(0, xa, sa), a1 = kv4_pair(0, xb, sb), a2 = kv4_pair(1, xa, sa), a3 = kv4_pair(1, xb, sb);
#pragma unroll
          for (int nt = 0; nt < NT; nt++) i4_mma(s[u][nt], a0, a1, a2, a3, qf[nt][w][2 * j], qf[nt][w][2 * j + 1]);
        }
      }
    }
    if constexpr (EDGE) {
#pragma unroll
      for (int u = 0; u < N; u++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int t = t0 + u * KV4_TOKENS + r + (e >> 1) * 8;
            if (t < k_lo[nt][e & 1] || t >= k_hi[nt][e & 1]) s[u][nt][e] = -INFINITY;
          }
    }
    // running maxima: moved only where a score outgrows them by more than a factor of 2^8 (no probability then overflows bf16, and
    // all of them shrink together otherwise), so most tiles need a vote and no exchange
    bool grow = false;
    float mt[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float x = fmaxf(s[0][nt][e], s[0][nt][e + 2]);
#pragma unroll
        for (int u = 1; u < N; u++) x = fmaxf(x, fmaxf(s[u][nt][e], s[u][nt][e + 2]));
        mt[nt][e] = x;
        grow |= x * p.scale_log2 > m[nt][e] + 8.f;
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float x = mt[nt][e];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const float now = fmaxf(m[nt][e], x * p.scale_log2), f = m[nt][e] == -INFINITY ? 0.f : i4_exp2(m[nt][e] - now);
          m[nt][e] = now;
          l[nt][e] *= f;
#pragma unroll
          for (int i = 0; i < MT; i++) {
            o[nt][i][e] *= f;
            o[nt][i][e + 2] *= f;
          }
        }
    }
    uint32_t pf[N][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const float n0 = m[nt][0] == -INFINITY ? 0.f : -m[nt][0], n1 = m[nt][1] == -INFINITY ? 0.f : -m[nt][1];
#pragma unroll
      for (int u = 0; u < N; u++) {
        const float p0 = i4_exp2(fmaf(s[u][nt][0], p.scale_log2, n0)), p1 = i4_exp2(fmaf(s[u][nt][1], p.scale_log2, n1));
        const float p2 = i4_exp2(fmaf(s[u][nt][2], p.scale_log2, n0)), p3 = i4_exp2(fmaf(s[u][nt][3], p.scale_log2, n1));
        l[nt][0] += p0 + p2;
        l[nt][1] += p1 + p3;
        // bf16 probabilities for the tensor cores (the sums above are of the fp32 ones): half a step of 2^-8, with either sign
        pf[u][nt][0] = i4_transpose(pack_bf16x2(p0, p1));
        pf[u][nt][1] = i4_transpose(pack_bf16x2(p2, p3));
      }
    }
    bool odd = false;                            // a scale that is no number
#pragma unroll
    for (int u = 0; u < N; u++) {
      const uint8_t* unit = vs + u * Cfg::UNIT;
      const uint32_t* sc = reinterpret_cast<const uint32_t*>(unit + kv4_scale(D, 2 * c, vg));
      uint32_t sw[2] = {sc[0], sc[4]};
      if constexpr (EDGE) {                      // tokens that no row sees weigh nothing, whatever lies in their place
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int t = t0 + u * KV4_TOKENS + 2 * c + 8 * i;
          if (t < lo || t >= hi) sw[i] &= 0xffff0000u;
          if (t + 1 < lo || t + 1 >= hi) sw[i] &= 0x0000ffffu;
          if ((sw[i] & 0x7f80u) == 0x7f80u) { sw[i] &= 0xffff0000u; odd = true; }
          if ((sw[i] & 0x7f800000u) == 0x7f800000u) { sw[i] &= 0x0000ffffu; odd = true; }
        }
      }
      const Kv4Scale sv[2] = {Kv4Scale(sw[0]), Kv4Scale(sw[1])};
      uint32_t x[2][2 * VX];                     // [tokens 2 c, + 8][two channels]: low bytes of a word, then its high ones
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const uint8_t* a = unit + kv4_value_word(D, 2 * c + 8 * i, r * (D / 8));
        uint32_t v[VX];
        if constexpr (VX == 4) {
          const uint4 e = *reinterpret_cast<const uint4*>(a);
          v[0] = e.x; v[1] = e.y; v[2] = e.z; v[3] = e.w;
        } else {
          const uint2 e = *reinterpret_cast<const uint2*>(a);
          v[0] = e.x; v[1] = e.y;
        }
#pragma unroll
        for (int w = 0; w < VX; w++) {
          x[i][2 * w] = v[w];
          x[i][2 * w + 1] = v[w] >> 8;
        }
      }
      // rows r of channel tile i: the lane's channel i, rows r + 8 its channel i + MT
#pragma unroll
      for (int i = 0; i < MT; i++) {
        const int j = i & 1, at = i >> 1, up = at + MT / 2;
        const uint32_t a0 = kv4_pair(j, x[0][at], sv[0]), a1 = kv4_pair(j, x[0][up], sv[0]);
        const uint32_t a2 = kv4_pair(j, x[1][at], sv[1]), a3 = kv4_pair(j, x[1][up], sv[1]);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) i4_mma(o[nt][i], a0, a1, a2, a3, pf[u][nt][0], pf[u][nt][1]);
      }
    }
    if (EDGE && __any_sync(0xffffffffu, odd)) {
      // values that are no numbers reach the rows that see them, and no others
      for (int i = 0; i < N * KV4_TOKENS; i++) {
        const int t = t0 + i;
        if (t < lo || t >= hi) continue;
        const uint16_t sc = *reinterpret_cast<const uint16_t*>(vs + (i / KV4_TOKENS) * Cfg::UNIT + kv4_scale(D, i % KV4_TOKENS, vg));
        if ((sc & 0x7f80u) != 0x7f80u) continue;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 2; e++)
            if (t >= k_lo[nt][e] && t < k_hi[nt][e])
#pragma unroll
              for (int j = 0; j < MT; j++) o[nt][j][e] = o[nt][j][e + 2] = __int_as_float(0x7fc00000);
      }
    }
  };
  auto inside = [&](int u, int n) { return u * KV4_TOKENS >= all_lo && (u + n) * KV4_TOKENS <= all_hi; };

  int stage = 0;
  uint32_t phase = 0;
  bool late = false;
  for (int u0 = first; u0 < last; u0 += U) {
    if (bad && u0 >= next) break;                // tiles from a bad page on were not fetched
    late = !__all_sync(0xffffffffu, mbar_wait(&bars[stage], phase, abort_word));
    if (late) break;
    const uint8_t* ks = ring + stage * Cfg::STAGE;
    const uint8_t* vs = ks + U * Cfg::UNIT;
    const int n = min(U, last - u0);
    if (n == U && inside(u0, U)) {
      tokens(std::integral_constant<int, U>(), std::false_type(), ks, vs, u0 * KV4_TOKENS);
    } else {
#pragma unroll 1
      for (int u = 0; u < n;) {
        if (n - u >= 2 && inside(u0 + u, 2)) {
          tokens(std::integral_constant<int, 2>(), std::false_type(), ks + u * Cfg::UNIT, vs + u * Cfg::UNIT, (u0 + u) * KV4_TOKENS);
          u += 2;
        } else {
          tokens(std::integral_constant<int, 1>(), std::true_type(), ks + u * Cfg::UNIT, vs + u * Cfg::UNIT, (u0 + u) * KV4_TOKENS);
          u++;
        }
      }
    }
    __syncwarp();                                // all lanes have read the stage
    if (next < last && !bad) issue(stage);
    if (++stage == Cfg::STAGES) {
      stage = 0;
      phase ^= 1;
    }
  }

  if (late) {                                    // copies still in flight land before the ring gets results, or is released
    const uint64_t t_start = globaltimer_ns();
    while (globaltimer_ns() - t_start < 50000ull) __nanosleep(1000);
  }
  // ---------------- join the warps: results into the rings' place
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      float x = l[nt][e];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      if (r == 0) {
        ms[warp * ROWS + nt * 8 + 2 * c + e] = m[nt][e];
        ls[warp * ROWS + nt * 8 + 2 * c + e] = x;
      }
    }
  if (bad && lane == 0) *bad_page = 1;
  float* res = (float*)ring;                     // [rows][D]
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      float* dst = res + (nt * 8 + 2 * c + e) * D + r * (D / 8);
#pragma unroll
      for (int i = 0; i < MT; i += 4) {
        *reinterpret_cast<float4*>(dst + i) = make_float4(o[nt][i][e], o[nt][i + 1][e], o[nt][i + 2][e], o[nt][i + 3][e]);
        *reinterpret_cast<float4*>(dst + MT + i) =
            make_float4(o[nt][i][e + 2], o[nt][i + 1][e + 2], o[nt][i + 2][e + 2], o[nt][i + 3][e + 2]);
      }
    }
  __syncthreads();
  if (threadIdx.x == 0 && p.status && (*abort_word != 0 || *bad_page != 0)) atomicExch(p.status, *bad_page ? B200_BAD_INDEX : *abort_word);
  float* block_o = (float*)i4_smem + ROWS * D;
  for (int it = threadIdx.x; it < rows * (D / 8); it += 32 * D4_WARPS) {
    const int i = it / (D / 8), ch = (it - i * (D / 8)) * 8;
    float top = ms[i];
#pragma unroll
    for (int w = 1; w < D4_WARPS; w++) top = fmaxf(top, ms[w * ROWS + i]);
    float sum = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < D4_WARPS; w++) {
      const float mw = ms[w * ROWS + i];
      if (mw == -INFINITY && ls[w * ROWS + i] == 0.f) continue;                // saw no key
      const float f = i4_exp2(mw - top);
      sum += ls[w * ROWS + i] * f;
      const float4* src = reinterpret_cast<const float4*>(i4_smem + w * Cfg::RING) + (i * D + ch) / 4;
      const float4 a = src[0], b = src[1];
      acc[0] += a.x * f; acc[1] += a.y * f; acc[2] += a.z * f; acc[3] += a.w * f;
      acc[4] += b.x * f; acc[5] += b.y * f; acc[6] += b.z * f; acc[7] += b.w * f;
    }
    const float inv = sum == 0.f ? 0.f : KV4_UNDO / sum;     // a row without keys: zeros
    const int tok = int4_div(row0 + i, p.G, p.g_inv), g = row0 + i - tok * p.G;
    if (p.cluster) {
      float4* dst = reinterpret_cast<float4*>(block_o + i * D + ch);
      dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      if (ch == 0) {
        block_m[i] = top;
        block_l[i] = sum;
      }
    } else if (p.parts == 1) {
      uint4 v;
      v.x = pack_bf16x2(acc[0] * inv, acc[1] * inv);
      v.y = pack_bf16x2(acc[2] * inv, acc[3] * inv);
      v.z = pack_bf16x2(acc[4] * inv, acc[5] * inv);
      v.w = pack_bf16x2(acc[6] * inv, acc[7] * inv);
      *reinterpret_cast<uint4*>(p.out + (long)(q_start + tok) * p.out_stride + (long)(h * p.G + g) * D + ch) = v;
    } else {
      const long at = ((long)(q_start + tok) * (p.Hkv * p.G) + h * p.G + g) * p.parts + part;
      float4* dst = reinterpret_cast<float4*>(p.part_o + at * D + ch);
      dst[0] = make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
      dst[1] = make_float4(acc[4] * inv, acc[5] * inv, acc[6] * inv, acc[7] * inv);
      if (ch == 0) p.part_lse[at] = sum == 0.f ? -INFINITY : top + log2f(sum);
    }
  }
  if (p.cluster) {
    // the parts' blocks form a cluster: each joins every parts-th piece of the rows out of all blocks' shared memory
    sg_cluster_sync();
    for (int it = part * 32 * D4_WARPS + threadIdx.x; it < rows * (D / 4); it += p.parts * 32 * D4_WARPS) {
      const int i = it / (D / 4), ch = (it - i * (D / 4)) * 4;
      // eight parts at a time, whose loads are under way together
      float top = -INFINITY, sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int q0 = 0; q0 < p.parts; q0 += 8) {
        float pm[8], pl[8], now = top;
        float4 po[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
          const int q = q0 + k;
          pm[k] = -INFINITY;
          pl[k] = 0.f;
          if (q < p.parts) {
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(pm[k]) : "r"(sg_map(smem_u32(block_m + i), q)) : "memory");
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(pl[k]) : "r"(sg_map(smem_u32(block_l + i), q)) : "memory");
            po[k] = sg_ld(sg_map(smem_u32(block_o + i * D + ch), q));
          }
          now = fmaxf(now, pm[k]);
        }
        if (q0 > 0 && top != -INFINITY) {
          const float f = i4_exp2(top - now);
          sum *= f;
          acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
        }
        top = now;
#pragma unroll
        for (int k = 0; k < 8; k++) {
          if (q0 + k >= p.parts || (pm[k] == -INFINITY && pl[k] == 0.f)) continue;     // saw no key
          const float f = i4_exp2(pm[k] - top);
          sum += pl[k] * f;
          acc.x += po[k].x * f; acc.y += po[k].y * f; acc.z += po[k].z * f; acc.w += po[k].w * f;
        }
      }
      const float inv = sum == 0.f ? 0.f : KV4_UNDO / sum;
      const int tok = int4_div(row0 + i, p.G, p.g_inv), g = row0 + i - tok * p.G;
      *reinterpret_cast<uint2*>(p.out + (long)(q_start + tok) * p.out_stride + (long)(h * p.G + g) * D + ch) =
          make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
    }
    sg_cluster_sync();                           // no block leaves while others read it
  }
}

// Parts of a (token, head) joined: sum 2^(lse_i - max) o_i / sum 2^(lse_i - max).  A warp each; tokens of listed sequences only.
template <int D>
__global__ void __launch_bounds__(128) attn_int4_join_kernel(const float* part_o, const float* part_lse, const int* cu, int num_seqs, int heads,
                                                             int parts, long rows, __nv_bfloat16* out, long out_stride) {
  const long at = (long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const long first = cu[0], end = cu[num_seqs];
  const long tok = first + at / heads;
  const int head = (int)(at % heads);
  if (at >= rows || tok < 0 || tok >= end || tok * heads >= rows) return;
  const float* lse = part_lse + (tok * heads + head) * parts;
  const float* o = part_o + (tok * heads + head) * parts * D;
  // a lane's weights: of parts lane and lane + 32
  const float x0 = lane < parts ? lse[lane] : -INFINITY, x1 = lane + 32 < parts ? lse[lane + 32] : -INFINITY;
  float top = warp_reduce_max(fmaxf(x0, x1));
  if (top == -INFINITY) top = 0.f;
  const float w0 = x0 == -INFINITY ? 0.f : i4_exp2(x0 - top), w1 = x1 == -INFINITY ? 0.f : i4_exp2(x1 - top);
  const uint32_t here0 = __ballot_sync(0xffffffffu, x0 != -INFINITY), here1 = __ballot_sync(0xffffffffu, x1 != -INFINITY);
  const float sum = warp_reduce_sum(w0 + w1);
  constexpr int V = D / 32;
  float acc[V] = {};
  for (int i0 = 0; i0 < parts; i0 += 8) {
    float a[8][V];
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const int i = i0 + k;
#pragma unroll
      for (int v = 0; v < V; v++) a[k][v] = 0.f;
      if ((i < 32 ? here0 >> i : here1 >> (i - 32)) & 1u) {      // others saw no key, and nothing was written
        if constexpr (V == 4) {
          const float4 x = reinterpret_cast<const float4*>(o + (long)i * D)[lane];
          a[k][0] = x.x; a[k][1] = x.y; a[k][2] = x.z; a[k][3] = x.w;
        } else {
          const float2 x = reinterpret_cast<const float2*>(o + (long)i * D)[lane];
          a[k][0] = x.x; a[k][1] = x.y;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const float f = __shfl_sync(0xffffffffu, i0 < 32 ? w0 : w1, (i0 + k) & 31);
#pragma unroll
      for (int v = 0; v < V; v++) acc[v] += a[k][v] * f;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint32_t* dst = reinterpret_cast<uint32_t*>(out + tok * out_stride + (long)head * D) + lane * (V / 2);
  dst[0] = pack_bf16x2(acc[0] * inv, acc[1] * inv);
  if constexpr (V == 4) dst[1] = pack_bf16x2(acc[2] * inv, acc[3] * inv);
}

template <int D, int NT>
static int launch_int4(Int4Params p, int max_rows, cudaStream_t stream) {
  using Cfg = Int4Cfg<D, NT>;
  cudaError_t e = allow_smem<attn_int4_kernel<D, NT>>(Cfg::SMEM);
  if (e != cudaSuccess) return (int)e;
  if (p.cluster && p.parts > 8) {                // more than every GPU of the architecture promises
    e = cudaFuncSetAttribute(attn_int4_kernel<D, NT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return (int)e;
  }
  p.row_blocks = (max_rows + Cfg::ROWS - 1) / Cfg::ROWS;
  const long x = (long)p.num_seqs * p.row_blocks;
  if (x > 0x7fffffffl || p.Hkv > 65535) return 9886;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)x, (unsigned)p.Hkv, (unsigned)p.parts);
  cfg.blockDim = dim3(32 * D4_WARPS);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = p.parts;
  cfg.attrs = &attr;
  cfg.numAttrs = p.cluster;
  e = cudaLaunchKernelEx(&cfg, attn_int4_kernel<D, NT>, p);
  return e != cudaSuccess ? (int)e : B200_CHECK_LAUNCH();
}

int int4_params(Int4Params* p, const Int4Args& a) {
  const int G = a.Hkv > 0 ? a.Hq / a.Hkv : 0;
  if (G < 1 || G * a.Hkv != a.Hq || (a.D != 64 && a.D != 128)) return 9883;
  if (a.block_size < KV4_TOKENS || a.block_size % KV4_TOKENS) return 9884;
  if ((a.q_stride & 7) || (a.out_stride & 7) || a.parts < 1 || a.parts > I4_PARTS) return 9885;
  *p = Int4Params{};
  p->q = (const __nv_bfloat16*)a.q;
  p->k_cache = (const uint8_t*)a.k_cache;
  p->v_cache = (const uint8_t*)a.v_cache;
  p->cu = a.cu;
  p->seq_lens = a.seq_lens;
  p->block_table = a.block_table;
  p->out = (__nv_bfloat16*)a.out;
  p->part_o = (float*)a.scratch;
  p->part_lse = p->part_o + a.q_rows * a.Hq * a.parts * a.D;
  p->q_stride = a.q_stride; p->out_stride = a.out_stride; p->table_stride = a.table_stride; p->num_blocks = a.num_blocks;
  p->q_rows = a.q_rows;
  p->num_seqs = a.num_seqs; p->max_blocks = a.max_blocks; p->block_size = a.block_size;
  p->G = G; p->Hkv = a.Hkv; p->parts = a.parts; p->causal = a.causal; p->window = a.window;
  const int upp = a.block_size / KV4_TOKENS;
  // what int4_div takes, and units times parts in 32 bits: tables of nearly 2^30 tokens (a sequence of that many takes 72 GiB a head of 64)
  if ((long)a.max_blocks * upp * upp > 0xffffffffl || (long)a.max_blocks * upp > 0xffffffffl / I4_PARTS) return 9888;
  p->g_inv = (uint32_t)((0x100000000ll + G - 1) / G);
  p->upp_inv = (uint32_t)((0x100000000ll + upp - 1) / upp);
  p->scale_log2 = a.scale * 1.4426950408889634f * KV4_UNDO;
  p->status = a.status;
  return 0;
}

int int4_join(const Int4Params& p, int D, long q_rows, cudaStream_t stream) {
  const int heads = p.G * p.Hkv;
  const long all = q_rows * heads;
  if ((all + 3) / 4 > 0x7fffffffl) return 9886;
  const unsigned blocks = (unsigned)((all + 3) / 4);
  if (D == 128) attn_int4_join_kernel<128><<<blocks, 128, 0, stream>>>(p.part_o, p.part_lse, p.cu, p.num_seqs, heads, p.parts, all, p.out, p.out_stride);
  else attn_int4_join_kernel<64><<<blocks, 128, 0, stream>>>(p.part_o, p.part_lse, p.cu, p.num_seqs, heads, p.parts, all, p.out, p.out_stride);
  return B200_CHECK_LAUNCH();
}

}  // namespace b200

using namespace b200;

// q [*, Hq, D] and out rows with token strides; cu [num_seqs + 1] their row numbers; max_q_len: no sequence has more new tokens.
// parts > 1: joined in a cluster (up to I4_CLUSTER), or, where scratch of (rows of q) x Hq x parts x (D + 1) floats is given, there.
B200_API int b200_attn_int4(const Int4Args* a) {
  if (a->num_seqs <= 0 || a->q_rows <= 0 || a->max_q_len <= 0) return 0;
  Int4Params p;
  int rc = int4_params(&p, *a);
  if (rc) return rc;
  const long rows = (long)a->max_q_len * p.G;
  if (rows * p.G > 0x7fffffffl) return 9886;
  p.cluster = p.parts > 1 && !a->scratch;
  if (p.cluster && p.parts > I4_CLUSTER) return 9885;
  if (a->D == 128) rc = rows <= 8 ? launch_int4<128, 1>(p, (int)rows, a->stream) : launch_int4<128, 2>(p, (int)rows, a->stream);
  else rc = rows <= 8 ? launch_int4<64, 1>(p, (int)rows, a->stream) : launch_int4<64, 2>(p, (int)rows, a->stream);
  return rc || p.parts == 1 || p.cluster ? rc : int4_join(p, a->D, a->q_rows, a->stream);
}
