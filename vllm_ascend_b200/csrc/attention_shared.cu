// Attention of a batch whose sequences share prefixes, on tcgen05: beams of one prompt, requests behind one system prompt.
//
//   out = (sum_p e^(s_p - m) v_p + sum_o e^(s_o - m) v_o) / (sum_p e^(s_p - m) + sum_o e^(s_o - m))
//
// over the keys p of a group's prefix and the keys o of the sequence itself.  All query rows of a group (new tokens times the G heads of
// a KV head) meet the prefix together, so it is read once a group instead of once a sequence; each sequence meets its own keys
// behind it.  Both are work of one kind: up to two tiles of 128 query rows against a range of a block table's keys.
//
// A plan kernel, once a step for all layers, lists that work (a base: rows, table row, keys), gives every KV head of it tiles + 1
// units of cost, and hands each block an equal stretch of all units, cut wherever it falls: stretches are found by arithmetic
// (unit y belongs to block ceil((y + 1) blocks / units) - 1), so nothing is counted at run time and results repeat bit for bit.  A block
// leaves, for every piece of work that it touches, unnormalised rows with their maximum and sum; slot h + block - first block
// of the base tells pieces apart.  A last kernel joins them.
//
//   warps 0..3, 4..7   softmax, one thread a query row; step s of a block belongs to group s mod 2
//   warp 8             TMA producer;  warp 9  MMA issuer
// Up to 128 rows (a group's beams, a sequence's own keys): the groups of warps take tiles of 128 keys in turn, each with scores and an
// output of its own (S0, S1, O0, O1 fill tensor memory), joined at the end of the piece.  128 x 128 scores take a group
// about 1.5 us, 64 KB of keys and values an SM's share of HBM 1.47: two groups keep the stream going.  Above 128 rows both groups work on
// every tile, each with 128 rows of its own.  Probabilities replace scores in tensor memory; warps whose 32 rows are empty skip them.
// Rows of V that no key of the range stands for are zeroed in shared memory where a product would read them (their
// probabilities are zero, but 0 x NaN is not); scores of such keys are masked whatever they are.
// All waits are bounded.
#include "common.cuh"

#include <mutex>
#include <string>
#include <unordered_map>

namespace b200 {

constexpr int SH_THREADS = 320;
constexpr int SH_HALF = 128 * 128;           // 128 rows x 64 bf16
constexpr int SH_ROWS = 256;                 // query rows of a base at most

struct SharedBase {
  int tok0, ntok;              // query tokens
  int table_row;               // whose pages
  int key_lo, key_hi;          // keys of the range
  int q_pos0;                  // position of token tok0 among them (behind key_hi: all see all)
  int tiles;                   // tiles of 128 keys, tile 0 at key_lo rounded down
  int cum;                     // units of cost in front of it
  int part_row;                // first row of its partial results
  int seg0;                    // block of its first tile
  int pad[2];
};

// plan: [0] units of cost, [1] bases, then block_first[blocks], tok_prefix[tokens], tok_own[tokens] (base of a token, -1 no keys, -2 no
// sequence), group_ctx[groups], bases
struct PlanArgs {
  const int* cu;               // [seqs + 1] first query row of each sequence
  const int* seq_lens;
  const int* group_starts;     // [groups + 1] first sequence of each group
  const int* prefix_lens;      // [groups]
  int* plan;
  int* status;
  cudaStream_t stream;
  int seqs, groups, tokens, G, Hkv, blocks, max_bases, bases_at;       // bases_at: ints in front of the bases
};

__device__ __forceinline__ int plan_group_ctx(const PlanArgs& a) { return 2 + a.blocks + 2 * a.tokens; }

// block that unit y of n falls to, and the first unit of block b
__device__ __forceinline__ int block_of(long y, long n, long blocks) { return (int)(((y + 1) * blocks + n - 1) / n - 1); }
__device__ __forceinline__ int first_unit(long b, long n, long blocks) { return (int)(b * n / blocks); }

// exclusive sum over the block's 1024 threads; all: the sum of all
__device__ __forceinline__ int block_scan(int v, int* part, int& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += t;
  }
  __syncthreads();
  if (lane == 31) part[warp] = x;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < 32; w++) {
    const int t = part[w];
    before += w < warp ? t : 0;
    all += t;
  }
  return before + x - v;
}

__global__ void __launch_bounds__(1024) shared_plan_kernel(const PlanArgs a) {
  __shared__ int part[32];
  __shared__ int bad;
  const int tid = threadIdx.x;
  int* head = a.plan;
  int* block_first = head + 2;
  int* tok_prefix = block_first + a.blocks;
  int* tok_own = tok_prefix + a.tokens;
  int* group_ctx = head + plan_group_ctx(a);
  SharedBase* bases = reinterpret_cast<SharedBase*>(head + a.bases_at);
  if (tid == 0) bad = 0;
  __syncthreads();
  for (int t = tid; t < a.tokens; t += 1024) tok_prefix[t] = -1, tok_own[t] = -2;
  for (int g = tid; g < a.groups; g += 1024) group_ctx[g] = 0x7fffffff;
  // sequences and groups in order, inside what the host counted; else nothing is planned
  bool wrong = false;
  for (int s = tid; s < a.seqs; s += 1024) wrong |= a.cu[s] < 0 || a.cu[s + 1] < a.cu[s] || a.cu[s + 1] > a.tokens;
  for (int g = tid; g < a.groups; g += 1024)
    wrong |= a.group_starts[g] < 0 || a.group_starts[g + 1] < a.group_starts[g] || a.group_starts[g + 1] > a.seqs;
  if (wrong) bad = 1;
  __syncthreads();
  if (bad) {
    if (tid == 0) {
      head[0] = head[1] = 0;
      if (a.status) atomicExch(a.status, B200_BAD_INDEX);
    }
    return;
  }
  auto group_of = [&](int s) -> int {            // -1: in none
    int lo = 0, hi = a.groups;                   // groups [0, lo) begin at or before s
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.group_starts[mid] <= s) lo = mid + 1; else hi = mid;
    }
    return lo > 0 && s < a.group_starts[lo] ? lo - 1 : -1;
  };
  // a prefix ends in front of the first new token of all its sequences
  for (int s = tid; s < a.seqs; s += 1024) {
    const int q = a.cu[s + 1] - a.cu[s], g = q > 0 ? group_of(s) : -1;
    if (g >= 0) atomicMin(&group_ctx[g], max(0, a.seq_lens[s] - q));
  }
  __syncthreads();
  auto prefix_of = [&](int g) -> int { return g < 0 ? 0 : max(0, min(a.prefix_lens[g], group_ctx[g])); };
  // bases: groups in front, then sequences
  const int per = 2 * (128 / a.G);               // tokens of a base
  int count = 0;
  for (int e0 = 0; e0 < a.groups + a.seqs; e0 += 1024) {
    const int e = e0 + tid;
    int tok = 0, ntok = 0, row = 0, lo = 0, hi = 0, ctx = 0x3fffffff;
    const bool group = e < a.groups;
    if (group) {
      row = a.group_starts[e];
      const int end = a.group_starts[e + 1];
      if (end > row) {
        hi = prefix_of(e);
        tok = a.cu[row];
        ntok = hi > 0 ? a.cu[end] - tok : 0;
      }
    } else if (e < a.groups + a.seqs) {
      row = e - a.groups;
      tok = a.cu[row];
      ntok = a.cu[row + 1] - tok;
      hi = a.seq_lens[row];
      ctx = hi - ntok;
      lo = ntok > 0 ? prefix_of(group_of(row)) : 0;
    }
    const int mine = (ntok + per - 1) / per;
    int all;
    int at = count + block_scan(mine, part, all);
    count += all;
    for (int i = 0; i < mine; i++, at++) {
      SharedBase b;
      b.tok0 = tok + i * per;
      b.ntok = min(per, ntok - i * per);
      b.table_row = row;
      b.key_lo = lo;
      b.q_pos0 = group ? ctx : ctx + i * per;
      b.key_hi = group ? hi : min(hi, b.q_pos0 + b.ntok);
      b.tiles = b.key_hi > lo ? ((b.key_hi + 127) >> 7) - (lo >> 7) : 0;
      b.cum = b.part_row = b.seg0 = b.pad[0] = b.pad[1] = 0;
      bases[at] = b;
      int* to = group ? tok_prefix : tok_own;
      for (int t = 0; t < b.ntok; t++) to[b.tok0 + t] = b.tiles > 0 ? at : -1;
    }
  }
  __syncthreads();
  // cost
  int units = 0;
  for (int i0 = 0; i0 < count; i0 += 1024) {
    const int i = i0 + tid;
    const int tiles = i < count ? bases[i].tiles : 0;
    int all;
    const int before = units + block_scan(tiles > 0 ? a.Hkv * (tiles + 1) : 0, part, all);
    if (i < count) bases[i].cum = before;
    units += all;
  }
  // blocks and partial rows of every base; every block has a unit, so the blocks that share a head's tiles leave rows without a gap
  const int blocks = min(a.blocks, units);
  int rows = 0;
  for (int i0 = 0; i0 < count; i0 += 1024) {
    const int i = i0 + tid;
    int need = 0, first = 0, tiles = 0;
    if (i < count && (tiles = bases[i].tiles) > 0) {
      const long cum = bases[i].cum, cost = (long)a.Hkv * (tiles + 1);
      first = block_of(cum + 1, units, blocks);
      const int last = block_of(cum + cost - 1, units, blocks);
      need = bases[i].ntok * a.G * (a.Hkv + last - first);
      for (int b = cum > 0 ? block_of(cum - 1, units, blocks) + 1 : 0; b <= last; b++) block_first[b] = i;
    }
    int all;
    const int before = rows + block_scan(need, part, all);
    if (i < count) bases[i].part_row = before, bases[i].seg0 = first;
    rows += all;
  }
  if (tid == 0) head[0] = units, head[1] = count;
}

// ---------------------------------------------------------------- attention
struct SharedParams {
  const int* plan;
  const int* block_table;
  long pitch;                  // ints between rows of the table
  int max_blocks, block_size, rows_per_load, piece;
  int G, Hkv, Hq, tpt;         // tpt: tokens of a tile of 128 rows
  int blocks, tokens, bases_at;
  float scale_log2;
  float* part_o;               // [partial rows, D]
  float2* part_ml;             // [partial rows] maximum (log2, scaled) and sum
  long num_blocks_total;
  int* status;
  __nv_bfloat16* out;
  long out_stride;
};

template <int D>
struct SharedCfg {
  static constexpr int NH = D / 64;
  static constexpr int TILE = NH * SH_HALF;              // bytes of 128 rows
  static constexpr int NK = D == 128 ? 2 : 3;
  static constexpr int NV = D == 128 ? 3 : 5;
  static constexpr int SMEM = (2 + NK + NV) * TILE + 1024 + 1024 + 512;
};

__device__ __forceinline__ float sh_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// pieces of work of a block, in order
struct Pieces {
  const SharedBase* bases;
  int count, i, h, Hkv, x0, x1, t0, t1;
  SharedBase b;

  __device__ __forceinline__ void load() {
    const int4* p = reinterpret_cast<const int4*>(bases + i);
    const int4 u = __ldg(p), v = __ldg(p + 1), w = __ldg(p + 2);
    b.tok0 = u.x; b.ntok = u.y; b.table_row = u.z; b.key_lo = u.w;
    b.key_hi = v.x; b.q_pos0 = v.y; b.tiles = v.z; b.cum = v.w;
    b.part_row = w.x; b.seg0 = w.y;
  }
  __device__ __forceinline__ bool start(const SharedParams& p) {
    const int units = __ldg(p.plan);
    count = __ldg(p.plan + 1);
    bases = reinterpret_cast<const SharedBase*>(p.plan + p.bases_at);
    Hkv = p.Hkv;
    const int blocks = min(p.blocks, units);
    if ((int)blockIdx.x >= blocks) return false;
    x0 = first_unit(blockIdx.x, units, blocks);
    x1 = first_unit(blockIdx.x + 1, units, blocks);
    i = __ldg(p.plan + 2 + blockIdx.x);
    load();
    h = (x0 - b.cum) / (b.tiles + 1);
    return settle();
  }
  // to the first piece from (i, h) on that has tiles in this block
  __device__ __forceinline__ bool settle() {
    while (true) {
      const int at = b.cum + h * (b.tiles + 1) + 1;       // unit of tile 0
      if (b.tiles > 0) {
        if (at >= x1) return false;
        t0 = max(0, x0 - at);
        t1 = min(b.tiles, x1 - at);
        if (t1 > t0) return true;
      }
      if (!step()) return false;
    }
  }
  __device__ __forceinline__ bool step() {
    if (b.tiles <= 0 || ++h == Hkv) {
      h = 0;
      if (++i >= count) return false;
      load();
    }
    return true;
  }
  __device__ __forceinline__ bool next() { return step() && settle(); }
};

// a cursor over tiles of a block's pieces
struct Tiles {
  Pieces p;
  bool more;
  int t;                       // tile of the piece's range
  int nsel;                    // query tiles
  uint32_t gt, qc;             // tiles and query tiles in front
  __device__ __forceinline__ void start(const SharedParams& a) {
    more = p.start(a);
    gt = qc = 0;
    enter(a);
  }
  __device__ __forceinline__ void enter(const SharedParams& a) {
    if (more) t = p.t0, nsel = p.b.ntok > a.tpt ? 2 : 1;
  }
  __device__ __forceinline__ void next(const SharedParams& a) {
    gt++;
    if (++t == p.t1) {
      qc += nsel;
      more = p.next();
      enter(a);
    }
  }
  // columns of the tile that are keys of the range
  __device__ __forceinline__ int base() const { return ((p.b.key_lo >> 7) + t) << 7; }
  __device__ __forceinline__ int c_lo() const { return max(0, p.b.key_lo - base()); }
  __device__ __forceinline__ int c_hi() const { return min(128, p.b.key_hi - base()); }
};

template <int D>
__global__ void __launch_bounds__(SH_THREADS, 1)
attn_shared_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_q4,
                   const __grid_constant__ CUtensorMap tmap_q1, const __grid_constant__ CUtensorMap tmap_k,
                   const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_kp,
                   const __grid_constant__ CUtensorMap tmap_vp, const SharedParams p) {
  using Cfg = SharedCfg<D>;
  constexpr int NH = Cfg::NH, NK = Cfg::NK, NV = Cfg::NV, TILE = Cfg::TILE;
  constexpr int O_COL = 256;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* Qs = smem;
  uint8_t* Ks = Qs + 2 * TILE;
  uint8_t* Vs = Ks + NK * TILE;
  float2* ml = (float2*)(Vs + NV * TILE);          // [128] of the group of warps that does not finish a piece
  uint64_t* q_full = (uint64_t*)(ml + 128);        // 2
  uint64_t* q_empty = q_full + 2;                  // 2
  uint64_t* k_full = q_empty + 2;                  // NK
  uint64_t* k_empty = k_full + NK;
  uint64_t* v_full = k_empty + NK;                 // NV
  uint64_t* v_empty = v_full + NV;
  uint64_t* s_full = v_empty + NV;                 // 2: scores of group w
  uint64_t* p_full = s_full + 2;                   // 2: its probabilities
  uint64_t* o_full = p_full + 2;                   // 2: its last product of a piece
  uint64_t* o_free = o_full + 2;                   // 2: its output has been read
  uint64_t* ml_full = o_free + 2;
  uint64_t* ml_empty = ml_full + 1;
  uint32_t* tmem_ptr = (uint32_t*)(ml_empty + 1);
  volatile int* abort_word = (volatile int*)(tmem_ptr + 1);
  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; b++) {
      mbar_init(&q_full[b], 1);
      mbar_init(&q_empty[b], 1);
      mbar_init(&s_full[b], 1);
      mbar_init(&p_full[b], 4);
      mbar_init(&o_full[b], 1);
      mbar_init(&o_free[b], 4);
    }
    for (int b = 0; b < NK; b++) {
      mbar_init(&k_full[b], 1);
      mbar_init(&k_empty[b], 1);
    }
    for (int b = 0; b < NV; b++) {
      mbar_init(&v_full[b], 1);
      mbar_init(&v_empty[b], 1);
    }
    mbar_init(ml_full, 4);
    mbar_init(ml_empty, 4);
    *abort_word = 0;
    mbar_fence_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_ptr, 512);
    tmem_relinquish();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = warp_uniform(*tmem_ptr);

  if (warp == 8) {
    // ------------------------------------------------------------ producer: K0 K1 V0 K2 V1 K3 ..., queries in front of a piece's first keys
    const int rpl = p.rows_per_load, parts = 128 / rpl, piece = p.piece;
    Tiles ck, cv;
    ck.start(p);
    cv.start(p);
    // lane i: page of part i of a tile; parts outside of the range take the nearest page inside
    auto load_blk = [&](const Tiles& c) -> int {
      if (!c.more || lane >= parts) return 0;
      const int key = min(max(c.base() + lane * rpl, c.p.b.key_lo), c.p.b.key_hi - 1), col = key / p.block_size;
      return col < p.max_blocks ? __ldg(p.block_table + (long)c.p.b.table_row * p.pitch + col) : -1;
    };
    auto load_tile = [&](const Tiles& c, int blk_mine, uint8_t* dst, uint64_t* fullb, const CUtensorMap* whole, const CUtensorMap* pieces) -> bool {
      const bool bad = __any_sync(0xffffffffu, lane < parts && (blk_mine < 0 || blk_mine >= p.num_blocks_total));
      if (bad) {
        *abort_word = B200_BAD_INDEX;
        return false;
      }
      const int base = c.base(), lo = c.c_lo(), hi = c.c_hi();
      const bool full = lo == 0 && hi == 128;
      const int rows = full ? rpl : piece, first = full ? 0 : lo / rows, end = full ? parts : (hi + rows - 1) / rows;
      if (elect_one()) mbar_expect_tx(fullb, (uint32_t)((end - first) * rows * 128 * NH));
      __syncwarp();
      for (int i = first; i < end; i++) {
        const int blk = __shfl_sync(0xffffffffu, blk_mine, i * rows / rpl);
        const int off = (base + i * rows) % p.block_size;
        if (elect_one())
#pragma unroll
          for (int hf = 0; hf < NH; hf++)
            tma_load_4d(dst + hf * SH_HALF + i * rows * 128, full ? whole : pieces, fullb, hf * 64, c.p.h, off, blk);
        __syncwarp();
      }
      return true;
    };
    auto load_k = [&](int blk) -> bool {
      const uint32_t st = ck.gt % NK;
      if (ck.t == ck.p.t0) {
        for (int s = 0; s < ck.nsel; s++) {
          const uint32_t q = ck.qc + s, b = q & 1;
          if (!mbar_wait(&q_empty[b], ((q >> 1) & 1u) ^ 1u, abort_word)) return false;
          const int tok = ck.p.b.tok0 + s * p.tpt, n = min(p.tpt, ck.p.b.ntok - s * p.tpt);
          const int box = n <= 1 ? 1 : (n <= 4 && p.tpt > 4 ? 4 : p.tpt);
          const CUtensorMap* tm = box == p.tpt ? &tmap_q : (box == 1 ? &tmap_q1 : &tmap_q4);
          if (elect_one()) {
            mbar_expect_tx(&q_full[b], (uint32_t)(box * p.G * 128 * NH));
#pragma unroll
            for (int hf = 0; hf < NH; hf++) tma_load_4d(Qs + b * TILE + hf * SH_HALF, tm, &q_full[b], hf * 64, 0, ck.p.h, tok);
          }
          __syncwarp();
        }
      }
      if (!mbar_wait(&k_empty[st], ((ck.gt / NK) & 1u) ^ 1u, abort_word)) return false;
      return load_tile(ck, blk, Ks + st * TILE, &k_full[st], &tmap_k, &tmap_kp);
    };
    int blk = load_blk(ck);
    for (int i = 0; i < 2 && ck.more; i++) {
      if (!load_k(blk)) goto done;
      ck.next(p);
      blk = load_blk(ck);
    }
    while (cv.more) {
      const uint32_t st = cv.gt % NV;
      const int blk_v = load_blk(cv);
      if (!mbar_wait(&v_empty[st], ((cv.gt / NV) & 1u) ^ 1u, abort_word)) goto done;
      if (!load_tile(cv, blk_v, Vs + st * TILE, &v_full[st], &tmap_v, &tmap_vp)) goto done;
      cv.next(p);
      if (ck.more) {
        if (!load_k(blk)) goto done;
        ck.next(p);
        blk = load_blk(ck);
      }
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ MMA issuer: S(0) S(1), then P V(s) and S(s + 2)
    if (elect_one()) {
      constexpr uint32_t idesc_s = make_idesc_f16(128, 128, true, false, false);
      constexpr uint32_t idesc_o = make_idesc_f16(128, D, true, false, true);
      const uint64_t dq0 = make_smem_desc(smem_u32(Qs), 16, 1024, kLayoutSw128), dk0 = make_smem_desc(smem_u32(Ks), 16, 1024, kLayoutSw128);
      const uint64_t dv0 = make_smem_desc(smem_u32(Vs), SH_HALF, 1024, kLayoutSw128);
      Tiles cs, co;
      cs.start(p);
      co.start(p);
      int sel_s = 0, sel_o = 0;                  // query tile of the tile
      uint32_t ss = 0, so = 0;                   // steps
      uint32_t oc[2] = {0, 0};                   // pieces that each output has had
      auto issue_s = [&]() -> bool {
        const uint32_t w = ss & 1, st = cs.gt % NK, q = cs.qc + sel_s, b = q & 1;
        if (cs.t == cs.p.t0 && !mbar_wait(&q_full[b], (q >> 1) & 1u, abort_word)) return false;
        if (sel_s == 0 && !mbar_wait(&k_full[st], (cs.gt / NK) & 1u, abort_word)) return false;
        tc_fence_after();
        const uint64_t dq = dq0 + (uint32_t)(b * (TILE >> 4)), dk = dk0 + (uint32_t)(st * (TILE >> 4));
#pragma unroll
        for (int kk = 0; kk < D / 16; kk++) {
          const uint32_t o = ((kk >> 2) * SH_HALF + (kk & 3) * 32) >> 4;
          umma_f16_ss(tmem_base + w * 128, dq + o, dk + o, idesc_s, kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[w]);
        if (cs.t == cs.p.t1 - 1) umma_commit(&q_empty[b]);
        if (++sel_s == cs.nsel) {
          umma_commit(&k_empty[st]);
          sel_s = 0;
          cs.next(p);
        }
        ss++;
        return true;
      };
      for (int i = 0; i < 2 && cs.more; i++)
        if (!issue_s()) goto done;
      while (co.more) {
        const uint32_t w = so & 1, st = co.gt % NV;
        if (!mbar_wait(&p_full[w], (so >> 1) & 1u, abort_word)) goto done;
        if (sel_o == 0 && !mbar_wait(&v_full[st], (co.gt / NV) & 1u, abort_word)) goto done;
        const int turn = co.nsel == 2 ? 1 : 2;   // tiles between two of a group of warps
        const bool fresh = co.t - co.p.t0 < turn, last = co.p.t1 - co.t <= turn;
        if (fresh && !mbar_wait(&o_free[w], (oc[w] & 1u) ^ 1u, abort_word)) goto done;
        tc_fence_after();
        const uint64_t dv = dv0 + (uint32_t)(st * (TILE >> 4));
        const int k0 = co.c_lo() >> 4, k1 = (co.c_hi() + 15) >> 4;
        for (int kk = k0; kk < k1; kk++)
          umma_f16_ts(tmem_base + O_COL + w * 128, tmem_base + w * 128 + kk * 8, dv + kk * 128, idesc_o, (!fresh || kk > k0) ? 1u : 0u);
        if (last) {
          umma_commit(&o_full[w]);
          oc[w]++;
        }
        if (++sel_o == co.nsel) {
          umma_commit(&v_empty[st]);
          sel_o = 0;
          co.next(p);
        }
        so++;
        if (cs.more && !issue_s()) goto done;
      }
    }
  } else {
    // ------------------------------------------------------------ softmax and results, group of warps w
    const uint32_t w = warp >> 2;
    const int row = (warp & 3) * 32 + lane, G = p.G;
    const int tok = row / G;
    const uint32_t t_lane = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_s = t_lane + w * 128, t_o = t_lane + O_COL;
    const float sl2 = p.scale_log2;
    constexpr float kRescale = 8.f;              // log2 by which the reference maximum may lag behind
    Pieces c;
    bool more = c.start(p);
    uint32_t s0 = 0, gt0 = 0, oc[2] = {0, 0}, mc = 0;
    while (more) {
      const int n = c.t1 - c.t0, nsel = c.b.ntok > p.tpt ? 2 : 1;
      const uint32_t off = (w ^ s0) & 1u;        // my first step of the piece
      const int first = nsel == 2 ? 0 : (int)off, turn = nsel == 2 ? 1 : 2;
      const int tok_first = nsel == 2 && off ? p.tpt : 0;
      const int nt = min(p.tpt, c.b.ntok - tok_first);
      const bool row_valid = tok < nt && tok < p.tpt;
      const bool warp_valid = (warp & 3) * 32 < nt * G;
      const int q_pos = c.b.q_pos0 + tok_first + tok;
      const int k_hi = min(c.b.key_hi, q_pos + 1), all_hi = min(c.b.key_hi, c.b.q_pos0 + tok_first + 1);
      float m = -INFINITY, l = 0.f;
      for (int i = first; i < n; i += turn) {
        const uint32_t step = nsel == 2 ? s0 + 2 * i + off : s0 + i, gt = gt0 + i;
        const int key0 = ((c.b.key_lo >> 7) + c.t0 + i) << 7;
        const int c_lo = max(0, c.b.key_lo - key0), c_hi = min(128, c.b.key_hi - key0);
        if (!mbar_wait(&s_full[w], (step >> 1) & 1u, abort_word)) goto done;
        tc_fence_after();
        if (warp_valid) {
          uint32_t sreg[128];
#pragma unroll
          for (int ch = 0; ch < 4; ch++)
            if (ch * 32 < c_hi && ch * 32 + 32 > c_lo) tmem_ld_32x32b_x32(t_s + ch * 32, sreg + ch * 32);
          tmem_ld_wait();
          if (c_lo > 0 || key0 + 128 > all_hi) {
#pragma unroll
            for (int j = 0; j < 128; j++)
              if (j < c_lo || key0 + j >= k_hi) sreg[j] = 0xff800000u;   // -inf
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int ch = 0; ch < 4; ch++)
            if (ch * 32 < c_hi && ch * 32 + 32 > c_lo) {
#pragma unroll
              for (int j = 0; j < 32; j += 8)
#pragma unroll
                for (int q = 0; q < 4; q++)
                  mx[q] = fmaxf(mx[q], fmaxf(__uint_as_float(sreg[ch * 32 + j + 2 * q]), __uint_as_float(sreg[ch * 32 + j + 2 * q + 1])));
            }
          const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          float alpha = 1.f;
          bool need = false;
          if (mt > m && (m == -INFINITY || (mt - m) * sl2 > kRescale)) {
            alpha = m == -INFINITY ? 0.f : sh_exp2((m - mt) * sl2);
            need = m != -INFINITY;               // a row without keys so far has zeros only
            m = mt;
          }
          l *= alpha;
          if (i > first && __any_sync(0xffffffffu, need && row_valid)) {
            const float a = need ? alpha : 1.f;
#pragma unroll 1
            for (int ch = 0; ch < D / 32; ch++) {
              uint32_t r[32];
              tmem_ld_32x32b_x32(t_o + w * 128 + ch * 32, r);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; j++) r[j] = __float_as_uint(__uint_as_float(r[j]) * a);
              tmem_st_32x32b_x32(t_o + w * 128 + ch * 32, r);
            }
          }
          const float nmb = m == -INFINITY ? 0.f : -m * sl2;
          float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ch = 0; ch < 4; ch++)
            if (ch * 32 < c_hi && ch * 32 + 32 > c_lo) {
              uint32_t pk[16];
#pragma unroll
              for (int j = 0; j < 16; j++) {
                const float p0 = sh_exp2(fmaf(__uint_as_float(sreg[ch * 32 + 2 * j]), sl2, nmb));
                const float p1 = sh_exp2(fmaf(__uint_as_float(sreg[ch * 32 + 2 * j + 1]), sl2, nmb));
                rs[(j & 1) * 2] += p0;
                rs[(j & 1) * 2 + 1] += p1;
                pk[j] = pack_bf16x2(p0, p1);     // the product takes bf16; the sum keeps 32 bits
              }
              tmem_st_32x32b_x16(t_s + ch * 16, pk);
            }
          l += (rs[0] + rs[1]) + (rs[2] + rs[3]);
          tmem_st_wait();
        }
        if ((c_lo & 15) || (c_hi & 15)) {        // rows of V beside the range that the product's steps of 16 keys reach
          if (nsel == 1 || off == 0) {
            const uint32_t st = gt % NV;
            if (!mbar_wait(&v_full[st], (gt / NV) & 1u, abort_word)) goto done;
            const int lo0 = c_lo & ~15, hi1 = (c_hi + 15) & ~15, nlo = c_lo - lo0, rows = nlo + hi1 - c_hi;
            for (int j = row; j < rows * 8 * NH; j += 128) {
              const int r = j / (8 * NH), x = j - r * 8 * NH, at = r < nlo ? lo0 + r : c_hi + r - nlo;
              *reinterpret_cast<uint4*>(Vs + st * TILE + (x >> 3) * SH_HALF + at * 128 + (x & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[w]);
      }
      // ---- the piece's rows
      const bool both = nsel == 1 && n > 1;
      const uint32_t finisher = both ? (s0 + n - 1) & 1u : w;
      if (both && finisher != w) {
        if (!mbar_wait(ml_empty, (mc & 1u) ^ 1u, abort_word)) goto done;
        ml[row] = make_float2(m, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(ml_full);
      } else if (nsel == 2 || both || off == 0) {
        if (!mbar_wait(&o_full[w], oc[w] & 1u, abort_word)) goto done;
        float a_own = 1.f, a_other = 0.f;
        if (both) {
          if (!mbar_wait(&o_full[w ^ 1], oc[w ^ 1] & 1u, abort_word)) goto done;
          if (!mbar_wait(ml_full, mc & 1u, abort_word)) goto done;
          const float2 o = ml[row];
          __syncwarp();
          if (lane == 0) mbar_arrive(ml_empty);
          const float top = fmaxf(m, o.x);
          if (top > -INFINITY) {
            a_own = sh_exp2((m - top) * sl2);
            a_other = sh_exp2((o.x - top) * sl2);
          }
          l = l * a_own + o.y * a_other;
          m = top;
        }
        tc_fence_after();
        if (warp_valid) {
          const long at = (long)c.b.part_row + (long)(c.h + (int)blockIdx.x - c.b.seg0) * (c.b.ntok * G) + tok_first * G + row;
          if (row_valid) p.part_ml[at] = make_float2(l != l && m == -INFINITY ? 0.f : m * sl2, l);      // scores without a number count
          float* dst = p.part_o + at * D;
#pragma unroll 1
          for (int ch = 0; ch < D / 32; ch++) {
            uint32_t r[32], x[32];
            tmem_ld_32x32b_x32(t_o + w * 128 + ch * 32, r);
            if (both) tmem_ld_32x32b_x32(t_o + (w ^ 1) * 128 + ch * 32, x);
            tmem_ld_wait();
            if (both) {
#pragma unroll
              for (int j = 0; j < 32; j++) r[j] = __float_as_uint(__uint_as_float(r[j]) * a_own + __uint_as_float(x[j]) * a_other);
            }
            if (row_valid) {
#pragma unroll
              for (int j = 0; j < 8; j++)
                reinterpret_cast<uint4*>(dst + ch * 32)[j] = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&o_free[w]);
          if (both) mbar_arrive(&o_free[w ^ 1]);
        }
      }
      if (nsel == 2 || both) {
        oc[0]++;
        oc[1]++;
      } else {
        oc[s0 & 1u]++;
      }
      mc += both;
      s0 += n * nsel;
      gt0 += n;
      more = c.next();
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
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// One warp a (token, head): pieces of the prefix and of the sequence's own keys, by their maxima and sums.
template <int D>
__global__ void __launch_bounds__(256) shared_join_kernel(const SharedParams p) {
  const int lane = threadIdx.x & 31;
  const long id = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int t = (int)(id / p.Hq), hq = (int)(id - (long)t * p.Hq);
  if (t >= p.tokens) return;
  const int units = __ldg(p.plan), blocks = min(p.blocks, units);
  const int* tok_base = p.plan + 2 + p.blocks;
  const int which[2] = {__ldg(tok_base + t), __ldg(tok_base + p.tokens + t)};
  if (which[1] == -2) return;                    // behind the last sequence: left as it is
  const SharedBase* bases = reinterpret_cast<const SharedBase*>(p.plan + p.bases_at);
  const int h = hq / p.G, g = hq - h * p.G;
  long at[2];
  int n[2], rows[2];
#pragma unroll
  for (int k = 0; k < 2; k++) {
    n[k] = 0;
    if (which[k] < 0) continue;
    const int4* q = reinterpret_cast<const int4*>(bases + which[k]);
    const int4 u = __ldg(q), v = __ldg(q + 1), x = __ldg(q + 2);
    const int first = v.w + h * (v.z + 1) + 1;   // unit of its first tile
    const int b0 = block_of(first, units, blocks), b1 = block_of(first + v.z - 1, units, blocks);
    rows[k] = u.y * p.G;
    at[k] = (long)x.x + (long)(h + b0 - x.y) * rows[k] + (t - u.x) * p.G + g;
    n[k] = b1 - b0 + 1;
  }
  float top = -INFINITY;
  for (int k = 0; k < 2; k++)
    for (int i = lane; i < n[k]; i += 32) top = fmaxf(top, p.part_ml[at[k] + (long)i * rows[k]].x);
  top = warp_reduce_max(top);
  constexpr int V = D / 32;
  float acc[V], sum = 0.f;
#pragma unroll
  for (int j = 0; j < V; j++) acc[j] = 0.f;
  if (top > -INFINITY) {
    for (int k = 0; k < 2; k++)
#pragma unroll 4
      for (int i = 0; i < n[k]; i++) {
        const long r = at[k] + (long)i * rows[k];
        const float2 e = p.part_ml[r];
        const float f = sh_exp2(e.x - top);
        sum += f * e.y;
        if constexpr (V == 4) {
          const float4 o = reinterpret_cast<const float4*>(p.part_o + r * D)[lane];
          acc[0] += f * o.x; acc[1] += f * o.y; acc[2] += f * o.z; acc[3] += f * o.w;
        } else {
          const float2 o = reinterpret_cast<const float2*>(p.part_o + r * D)[lane];
          acc[0] += f * o.x; acc[1] += f * o.y;
        }
      }
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  __nv_bfloat16* dst = p.out + (long)t * p.out_stride + (long)hq * D + lane * V;
  if constexpr (V == 4)
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  else
    *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(acc[0] * inv, acc[1] * inv);
}

// ---------------------------------------------------------------- host
struct SharedArgs {
  const void* q;
  const void* k_cache;
  const void* v_cache;
  const int* plan;
  const int* block_table;
  float* parts;                // [rows, D + 2]: outputs, then maxima and sums
  void* out;
  int* status;
  cudaStream_t stream;
  long q_stride, T, num_blocks, pitch, out_stride, part_rows;
  long block_stride, token_stride, head_stride;      // of the caches, in elements
  float scale;
  int block_size, max_blocks, Hq, Hkv, D, blocks, tokens, bases_at;
};

static int shared_tmap(CUtensorMap* out, const void* base, const uint64_t* dims, const uint64_t* strides, const uint32_t* box) {
  static std::unordered_map<std::string, CUtensorMap> map;
  static std::mutex mu;
  char key[80];
  memcpy(key, &base, 8);
  memcpy(key + 8, dims, 32);
  memcpy(key + 40, strides, 24);
  memcpy(key + 64, box, 16);
  std::string k(key, 80);
  std::lock_guard<std::mutex> g(mu);
  auto it = map.find(k);
  if (it != map.end()) {
    *out = it->second;
    return 0;
  }
  const int rc = make_tmap(out, base, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  if (map.size() > 4096) map.clear();
  map.emplace(std::move(k), *out);
  return 0;
}

template <int D>
static int launch_shared(const CUtensorMap* tm, const SharedParams& p, cudaStream_t stream) {
  const cudaError_t e = allow_smem<&attn_shared_kernel<D>>(SharedCfg<D>::SMEM);
  if (e != cudaSuccess) return (int)e;
  attn_shared_kernel<D><<<p.blocks, SH_THREADS, SharedCfg<D>::SMEM, stream>>>(tm[0], tm[1], tm[2], tm[3], tm[4], tm[5], tm[6], p);
  const int rc = B200_CHECK_LAUNCH();
  if (rc) return rc;
  const long warps = (long)p.tokens * p.Hq;
  shared_join_kernel<D><<<(unsigned)((warps + 7) / 8), 256, 0, stream>>>(p);
  return B200_CHECK_LAUNCH();
}

}  // namespace b200

B200_API int b200_shared_plan(const b200::PlanArgs* args) {
  using namespace b200;
  const PlanArgs& a = *args;
  if (a.seqs < 0 || a.groups < 0 || a.tokens < 0 || a.G < 1 || a.G > 128 || a.Hkv < 1 || a.blocks < 1) return 9950;
  const int per = 2 * (128 / a.G);
  if ((long)a.max_bases < (long)a.groups + a.seqs + 2 * ((long)a.tokens / per) || (a.bases_at & 3) ||
      a.bases_at < 2 + a.blocks + 2 * a.tokens + a.groups || ((uintptr_t)a.plan & 15))
    return 9951;
  shared_plan_kernel<<<1, 1024, 0, a.stream>>>(a);
  return B200_CHECK_LAUNCH();
}

B200_API int b200_attn_shared(const b200::SharedArgs* args) {
  using namespace b200;
  const SharedArgs& a = *args;
  if (a.T <= 0 || a.tokens <= 0) return 0;
  const int bs = a.block_size;
  if (a.Hkv < 1 || a.Hq % a.Hkv || a.Hq / a.Hkv > 128 || (a.D != 64 && a.D != 128) || a.tokens > a.T) return 9955;
  if (bs < 8 || (bs < 128 && 128 % bs) || (bs > 128 && bs % 128)) return 9956;
  if ((a.q_stride & 7) || (a.out_stride & 7) || ((uintptr_t)a.q & 15) || ((uintptr_t)a.out & 15) || ((uintptr_t)a.k_cache & 15) ||
      ((uintptr_t)a.v_cache & 15) || (a.block_stride & 7) || (a.token_stride & 7) || (a.head_stride & 7))
    return 9957;
  const int G = a.Hq / a.Hkv, tpt = 128 / G;
  // what the pieces of a plan of these sizes have room for
  if (a.part_rows < 2L * a.tokens * a.Hq + (long)a.blocks * SH_ROWS) return 9958;
  CUtensorMap tm[7];
  {
    const uint64_t dims[4] = {(uint64_t)a.D, (uint64_t)G, (uint64_t)a.Hkv, (uint64_t)a.T};
    const uint64_t str[3] = {(uint64_t)a.D * 2, (uint64_t)G * a.D * 2, (uint64_t)a.q_stride * 2};
    const uint32_t n[3] = {(uint32_t)tpt, (uint32_t)(tpt < 4 ? tpt : 4), 1};
    for (int i = 0; i < 3; i++) {
      const uint32_t box[4] = {64, (uint32_t)G, 1, n[i]};
      const int rc = shared_tmap(&tm[i], a.q, dims, str, box);
      if (rc) return rc;
    }
  }
  const int rpl = bs < 128 ? bs : 128, piece = rpl < 32 ? rpl : 32;
  for (int i = 0; i < 4; i++) {
    const uint64_t dims[4] = {(uint64_t)a.D, (uint64_t)a.Hkv, (uint64_t)bs, (uint64_t)a.num_blocks};
    const uint64_t str[3] = {(uint64_t)a.head_stride * 2, (uint64_t)a.token_stride * 2, (uint64_t)a.block_stride * 2};
    const uint32_t box[4] = {64, 1, (uint32_t)(i < 2 ? rpl : piece), 1};
    const int rc = shared_tmap(&tm[3 + i], i & 1 ? a.v_cache : a.k_cache, dims, str, box);
    if (rc) return rc;
  }
  SharedParams p;
  p.plan = a.plan;
  p.block_table = a.block_table;
  p.pitch = a.pitch;
  p.max_blocks = a.max_blocks;
  p.block_size = bs;
  p.rows_per_load = rpl;
  p.piece = piece;
  p.G = G; p.Hkv = a.Hkv; p.Hq = a.Hq; p.tpt = tpt;
  p.blocks = a.blocks;
  p.tokens = a.tokens;
  p.bases_at = a.bases_at;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.part_o = a.parts;
  p.part_ml = (float2*)(a.parts + a.part_rows * a.D);
  p.num_blocks_total = a.num_blocks;
  p.status = a.status;
  p.out = (__nv_bfloat16*)a.out;
  p.out_stride = a.out_stride;
  return a.D == 64 ? launch_shared<64>(tm, p, a.stream) : launch_shared<128>(tm, p, a.stream);
}
