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
//   warps 8, 10        TMA producers of queries and keys, of values;  warp 9  MMA issuer
// Up to 128 rows (a group's beams, a sequence's own keys): the groups of warps take tiles of 128 keys in turn, each with scores and an
// output of its own (S0, S1, O0, O1 fill tensor memory) and results of its own.  128 x 128 scores take a group
// about 1.5 us, 64 KB of keys and values an SM's share of HBM 1.47: two groups keep the stream going.  Above 128 rows both groups work on
// every tile, each with 128 rows of its own.  Probabilities replace scores in tensor memory; warps whose 32 rows are empty skip them.
// Rows of V that no key of the range stands for are zeroed in shared memory where a product would read them (their
// probabilities are zero, but 0 x NaN is not); scores of such keys are masked whatever they are.
// All waits are bounded.
// Bound by HBM for long prefixes: 8 beams over 60000 keys (64 heads on 8 of 128, pages of 128) 57 us, 4.5 TB/s with beginning, end and join, which take
// 10 us of every call; 16 prompts of 8 beams over 2000 keys, 32 heads on 8, 50 us (128 requests read by themselves: 128).  Many requests behind one prompt are bound by
// their own keys: 192 over 2048 and 900 130 us, 5.4 TB/s.  Few keys are bound by the chain of a block's first tile, its results and the join: 14 us.
#include "common.cuh"

#include <mutex>
#include <string.h>
#include <unordered_map>

namespace b200 {

constexpr int SH_THREADS = 352;
constexpr int SH_HALF = 128 * 128;           // 128 rows x 64 bf16
constexpr int SH_ROWS = 256;                 // query rows of a base at most

struct SharedBase {
  int tok0, ntok;              // query tokens
  int table_row;               // whose pages
  int key_lo, key_hi;          // keys of the range
  int q_pos0;                  // position of token tok0 among them (behind key_hi: all see all)
  int tiles;                   // tiles of 128 keys, tile 0 at key_lo rounded down
  int weight;                  // units of a tile
  int cum;                     // units of cost in front of it
  int part_row;                // first row of its partial results
  int seg0;                    // block of its first tile
  int pad;
};

// What a tile of 128 keys, one for two query tiles (the softmax of twice the rows on the same schedulers) and the begin and end of a piece cost.  A piece
// of 256 rows loads and leaves two query tiles: counted like one of 128, blocks with many such pieces were late (192 requests behind 128 keys 183 us, 127).
constexpr int COST_TILE = 4, COST_PAIR = 9;
constexpr unsigned long long MOST_UNITS = 1ull << 30;
__host__ __device__ __forceinline__ constexpr int cost_piece(int weight) { return weight == COST_PAIR ? 13 : 4; }

// plan: [0] units of cost, [1] bases, [2] blocks with work, then block_first[blocks] and block_unit[blocks + 1] (base and unit that a block begins
// with), tok_prefix[tokens], tok_own[tokens] (base of a token, -1 no keys, -2 no sequence), group_ctx[groups], bases, and for every base and
// head the first row and the number of its partial results
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

constexpr int PLAN_HEAD = 3;
__host__ __device__ __forceinline__ int plan_tokens_at(int blocks) { return PLAN_HEAD + 2 * blocks + 1; }
__host__ __device__ __forceinline__ int plan_heads_at(int bases_at, int max_bases) {
  return bases_at + max_bases * (int)(sizeof(SharedBase) / 4);
}

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
  __shared__ unsigned long long all_units;
  const int tid = threadIdx.x;
  int* head = a.plan;
  int* block_first = head + PLAN_HEAD;
  int* block_unit = block_first + a.blocks;
  int* tok_prefix = head + plan_tokens_at(a.blocks);
  int* tok_own = tok_prefix + a.tokens;
  int* group_ctx = tok_own + a.tokens;
  SharedBase* bases = reinterpret_cast<SharedBase*>(head + a.bases_at);
  int2* heads = reinterpret_cast<int2*>(head + plan_heads_at(a.bases_at, a.max_bases));
  if (tid == 0) bad = 0, all_units = 0;
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
      head[0] = head[1] = head[2] = 0;
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
      b.tiles = b.key_hi > lo ? (int)(((unsigned)b.key_hi + 127) >> 7) - (lo >> 7) : 0;
      b.weight = b.ntok > per / 2 ? COST_PAIR : COST_TILE;
      b.cum = b.part_row = b.seg0 = b.pad = 0;
      bases[at] = b;
      int* to = group ? tok_prefix : tok_own;
      for (int t = 0; t < b.ntok; t++) to[b.tok0 + t] = b.tiles > 0 ? at : -1;
    }
  }
  __syncthreads();
  // Cost: units are counted in 32 bits.  What a cache can hold stays far below (180 GB are 50 million units); lengths that are none do not.
  unsigned long long mine = 0;
  for (int i = tid; i < count; i += 1024)
    if (bases[i].tiles > 0) mine += (unsigned long long)a.Hkv * ((long)bases[i].tiles * bases[i].weight + cost_piece(bases[i].weight));
  atomicAdd(&all_units, mine);
  __syncthreads();
  if (all_units > MOST_UNITS) {
    for (int t = tid; t < a.tokens; t += 1024) tok_prefix[t] = -1, tok_own[t] = -2;
    if (tid == 0) {
      head[0] = head[1] = head[2] = 0;
      if (a.status) atomicExch(a.status, B200_BAD_INDEX);
    }
    return;
  }
  int units = 0;
  for (int i0 = 0; i0 < count; i0 += 1024) {
    const int i = i0 + tid;
    const int tiles = i < count ? bases[i].tiles : 0;
    int all;
    const int before = units + block_scan(tiles > 0 ? a.Hkv * (tiles * bases[i].weight + cost_piece(bases[i].weight)) : 0, part, all);
    if (i < count) bases[i].cum = before;
    units += all;
  }
  // Blocks and partial rows of every base.  A block has as many units as a tile at least, so those from the one of a head's first tile to the one
  // of its last all have tiles of it, and their rows leave no gap.
  bool pairs = false;
  for (int i = tid; i < count; i += 1024) pairs |= bases[i].tiles > 0 && bases[i].weight == COST_PAIR;
  const int blocks = min(a.blocks, units / (__syncthreads_or(pairs) ? COST_PAIR : COST_TILE));
  int rows = 0;
  for (int i0 = 0; i0 < count; i0 += 1024) {
    const int i = i0 + tid;
    int need = 0, first = 0, tiles = 0;
    if (i < count && (tiles = bases[i].tiles) > 0) {
      const SharedBase b = bases[i];
      const long cum = b.cum, head_cost = (long)tiles * b.weight + cost_piece(b.weight), cost = a.Hkv * head_cost;
      first = block_of(cum + cost_piece(b.weight), units, blocks);
      const int last = block_of(cum + cost - b.weight, units, blocks);
      // up to 128 rows, each group of warps leaves results of its own
      need = b.ntok * a.G * (a.Hkv + last - first) * (b.weight == COST_PAIR ? 1 : 2);
      const int end = block_of(cum + cost - 1, units, blocks);
      for (int c = cum > 0 ? block_of(cum - 1, units, blocks) + 1 : 0; c <= end; c++) block_first[c] = i;
    }
    int all;
    const int before = rows + block_scan(need, part, all);
    if (i < count) bases[i].part_row = before, bases[i].seg0 = first;
    rows += all;
  }
  for (int c = tid; c <= blocks; c += 1024) block_unit[c] = blocks > 0 ? first_unit(c, units, blocks) : 0;
  __syncthreads();
  for (int j = tid; j < count * a.Hkv; j += 1024) {
    const int i = j / a.Hkv, h = j - i * a.Hkv;
    const SharedBase b = bases[i];
    if (b.tiles <= 0) continue;
    const long at = b.cum + (long)h * (b.tiles * b.weight + cost_piece(b.weight)) + cost_piece(b.weight);       // unit of the first tile
    const int b0 = block_of(at, units, blocks), b1 = block_of(at + (b.tiles - 1) * b.weight, units, blocks);
    const int slots = b.weight == COST_PAIR ? 1 : 2;
    heads[j] = make_int2(b.part_row + (h + b0 - b.seg0) * slots * b.ntok * a.G, (b1 - b0 + 1) * slots);
  }
  if (tid == 0) head[0] = units, head[1] = count, head[2] = blocks;
}

// ---------------------------------------------------------------- attention
struct SharedParams {
  const int* plan;
  const int* block_table;
  long pitch;                  // ints between rows of the table
  int max_blocks, block_size, page_shift, rows_per_load, piece;        // page_shift: log2 of the block size, -1: no power of two
  int G, Hkv, Hq, tpt;         // tpt: tokens of a tile of 128 rows
  int blocks, tokens, bases_at, heads_at;
  int rows;                    // of q and out
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
  static constexpr int SMEM = (2 + NK + NV) * TILE + 384;        // of 228 KB, what a join's block needs stays free (each takes 1 KB more)
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
    b.key_hi = v.x; b.q_pos0 = v.y; b.tiles = v.z; b.weight = v.w;
    b.cum = w.x; b.part_row = w.y; b.seg0 = w.z;
  }
  __device__ __forceinline__ bool start(const SharedParams& p) {
    const int* at = p.plan + PLAN_HEAD + blockIdx.x;
    const int blocks = __ldg(p.plan + 2);
    i = __ldg(at);
    x0 = __ldg(at + p.blocks);
    x1 = __ldg(at + p.blocks + 1);
    count = __ldg(p.plan + 1);
    bases = reinterpret_cast<const SharedBase*>(p.plan + p.bases_at);
    Hkv = p.Hkv;
    if ((int)blockIdx.x >= blocks) return false;
    load();
    h = (x0 - b.cum) / (b.tiles * b.weight + cost_piece(b.weight));
    return settle();
  }
  // to the first piece from (i, h) on that has tiles in this block: a tile belongs to the block of its first unit
  __device__ __forceinline__ bool settle() {
    while (true) {
      if (b.tiles > 0) {
        const int at = b.cum + h * (b.tiles * b.weight + cost_piece(b.weight)) + cost_piece(b.weight);       // unit of tile 0
        if (at >= x1) return false;
        t0 = x0 > at ? (x0 - at + b.weight - 1) / b.weight : 0;
        t1 = min(b.tiles, (x1 - at + b.weight - 1) / b.weight);
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
attn_shared_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_q64,
                   const __grid_constant__ CUtensorMap tmap_q4, const __grid_constant__ CUtensorMap tmap_q1, const __grid_constant__ CUtensorMap tmap_k,
                   const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_kp,
                   const __grid_constant__ CUtensorMap tmap_vp, const SharedParams p) {
  using Cfg = SharedCfg<D>;
  constexpr int NH = Cfg::NH, NK = Cfg::NK, NV = Cfg::NV, TILE = Cfg::TILE;
  constexpr int O_COL = 256;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  extern __shared__ __align__(1024) uint8_t smem[];          // there is no other shared memory: it begins where the system's first KB ends
  if (smem_u32(smem) & 1023) {
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, B200_OVERFLOW);
    return;
  }
  uint8_t* Qs = smem;
  uint8_t* Ks = Qs + 2 * TILE;
  uint8_t* Vs = Ks + NK * TILE;
  uint64_t* q_full = (uint64_t*)(Vs + NV * TILE);  // 2
  uint64_t* q_empty = q_full + 2;                  // 2
  uint64_t* k_full = q_empty + 2;                  // NK
  uint64_t* k_empty = k_full + NK;
  uint64_t* v_full = k_empty + NK;                 // NV
  uint64_t* v_empty = v_full + NV;
  uint64_t* s_full = v_empty + NV;                 // 2: scores of group w
  uint64_t* p_full = s_full + 2;                   // 2: its probabilities
  uint64_t* o_full = p_full + 2;                   // 2: its last product of a piece
  uint64_t* o_free = o_full + 2;                   // 2: its output has been read
  int* pages = (int*)(o_free + 2);                 // 16 of each producer
  uint32_t* tmem_ptr = (uint32_t*)(pages + 32);
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
  // the join may take its place beside these blocks, all of them running by then, and find its rows; it waits for their end before it reads results
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp == 8 || warp == 10) {
    // ------------------------------------------------------------ producers: warp 8 queries and keys, warp 10 values; one thread of each walks the
    // loop (see warp_uniform).  One for both took 1.3 us a tile, about what the bytes take.
    if (elect_one()) {
      const bool values = warp == 10;
      const int rpl = p.rows_per_load, parts = 128 / rpl, depth = values ? NV : NK;
      const CUtensorMap* whole = values ? &tmap_v : &tmap_k;
      const CUtensorMap* pieces = values ? &tmap_vp : &tmap_kp;
      uint8_t* stages = values ? Vs : Ks;
      uint64_t* full_bars = values ? v_full : k_full;
      uint64_t* empty_bars = values ? v_empty : k_empty;
      Tiles c;
      c.start(p);
      // Pages of a tile's parts go to shared memory while the tile in front is waited for; parts outside of the range take the nearest page inside.
      // Loops stay rolled: what all roles execute a tile has to stay in the instruction caches (60000 keys: 54 us a block unrolled, 45 rolled).
      int* my_pages = pages + (values ? 16 : 0);
      auto fetch_pages = [&]() {
        const int* row = p.block_table + (long)c.p.b.table_row * p.pitch;
        const int base = c.base();
        if (p.page_shift >= 0 && c.c_lo() == 0 && c.c_hi() == 128 && (base + 127) >> p.page_shift < p.max_blocks) {
          row += base >> p.page_shift;
#pragma unroll 2
          for (int i = 0; i < parts; i++)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(my_pages + i)), "l"(row + i) : "memory");
          return;
        }
#pragma unroll 1
        for (int i = 0, key = base; i < parts; i++, key += rpl) {
          const int near = min(max(key, c.p.b.key_lo), c.p.b.key_hi - 1);
          const int col = p.page_shift >= 0 ? near >> p.page_shift : near / p.block_size;
          if (col < p.max_blocks) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(my_pages + i)), "l"(row + col) : "memory");
          else my_pages[i] = -1;
        }
      };
      if (c.more) fetch_pages();
      uint32_t st = 0, ph = 1;
      while (c.more) {
        if (!values && c.t == c.p.t0) {
          const bool twice = c.p.b.ntok * p.G <= 64;       // the second group of warps finds the rows 64 further on
#pragma unroll 1
          for (int s = 0; s < c.nsel; s++) {
            const uint32_t q = c.qc + s, b = q & 1;
            if (!mbar_wait(&q_empty[b], ((q >> 1) & 1u) ^ 1u, abort_word)) goto done;
            const int tok = c.p.b.tok0 + s * p.tpt, n = min(p.tpt, c.p.b.ntok - s * p.tpt);
            int box = p.tpt;                     // tokens of the copy
            const CUtensorMap* tm = &tmap_q;
            if (n == 1) box = 1, tm = &tmap_q1;
            else if (n <= 4 && p.G <= 16) box = 4, tm = &tmap_q4;
            else if (twice) box = 64 / p.G, tm = &tmap_q64;
            mbar_expect_tx(&q_full[b], (uint32_t)(box * p.G * 128 * NH * (twice ? 2 : 1)));
#pragma unroll 1
            for (int i = 0; i < (twice ? 2 : 1); i++)
#pragma unroll
              for (int hf = 0; hf < NH; hf++)
                tma_load_4d(Qs + b * TILE + hf * SH_HALF + i * 64 * 128, tm, &q_full[b], hf * 64, 0, c.p.h, tok);
          }
        }
        if (!mbar_wait(&empty_bars[st], ph, abort_word)) goto done;
        asm volatile("cp.async.wait_all;" ::: "memory");
        const int base = c.base(), lo = c.c_lo(), hi = c.c_hi();
        uint8_t* dst = stages + st * TILE;
        bool bad = false;                        // copies of pages out of range read zeros
        if (lo == 0 && hi == 128) {
          mbar_expect_tx(&full_bars[st], TILE);
          const int off = parts > 1 ? 0 : (p.page_shift >= 0 ? base & (p.block_size - 1) : base % p.block_size);
#pragma unroll 2
          for (int i = 0; i < parts; i++, dst += rpl * 128) {
            const int page = my_pages[i];
            bad |= (uint32_t)page >= (uint32_t)p.num_blocks_total;
#pragma unroll
            for (int hf = 0; hf < NH; hf++) tma_load_4d(dst + hf * SH_HALF, whole, &full_bars[st], hf * 64, c.p.h, off, page);
          }
        } else {
          const int rows = p.piece, end = (hi + rows - 1) / rows;
          mbar_expect_tx(&full_bars[st], (uint32_t)((end - lo / rows) * rows * 128 * NH));
#pragma unroll 1
          for (int i = lo / rows; i < end; i++) {
            const int page = my_pages[i * rows / rpl];
            const int off = p.page_shift >= 0 ? (base + i * rows) & (p.block_size - 1) : (base + i * rows) % p.block_size;
            bad |= (uint32_t)page >= (uint32_t)p.num_blocks_total;
#pragma unroll
            for (int hf = 0; hf < NH; hf++)
              tma_load_4d(dst + hf * SH_HALF + i * rows * 128, pieces, &full_bars[st], hf * 64, c.p.h, off, page);
          }
        }
        if (bad) {
          *abort_word = B200_BAD_INDEX;
          goto done;
        }
        if (++st == (uint32_t)depth) st = 0, ph ^= 1u;
        c.next(p);
        if (c.more) fetch_pages();
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
    const int lane_row = (warp & 3) * 32 + lane, G = p.G;
    const uint32_t t_lane = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_s = t_lane + w * 128, t_o = t_lane + O_COL;
    const float sl2 = p.scale_log2;
    constexpr float kRescale = 8.f;              // log2 by which the reference maximum may lag behind
    Pieces c;
    bool more = c.start(p);
    uint32_t s0 = 0, gt0 = 0, oc = 0;            // steps, tiles and pieces of mine in front
    while (more) {
      const int n = c.t1 - c.t0, nsel = c.b.ntok > p.tpt ? 2 : 1;
      const uint32_t off = (w ^ s0) & 1u;        // my first step of the piece
      const int first = nsel == 2 ? 0 : (int)off, turn = nsel == 2 ? 1 : 2;
      const int tok_first = nsel == 2 && off ? p.tpt : 0;
      const int nt = min(p.tpt, c.b.ntok - tok_first), rows = nt * G;
      // up to 64 rows: the second group's are 64 lanes further on, so that all four schedulers have a warp with rows
      const int shift = nsel == 1 && rows <= 64 && w == 1 ? 64 : 0, row = lane_row - shift, tok = row / G;
      const bool row_valid = row >= 0 && row < rows;
      const bool warp_valid = (warp & 3) * 32 >= shift && (warp & 3) * 32 - shift < rows;
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
          // Scores are read twice, for the maximum and for the exponentials, 32 columns at a time: held, the 128 of a row spilled (three warps
          // of a scheduler have 168 registers a thread) and a tile took 4.6 us.
          const bool masked = c_lo > 0 || key0 + 128 > all_hi;
          const int ch0 = c_lo >> 5, ch1 = (c_hi + 31) >> 5;
          auto hide = [&](int ch, uint32_t* x) {
            if (masked) {                        // columns of 32 that the row sees
              const int lo = c_lo - ch * 32, hi = k_hi - key0 - ch * 32;
              const uint32_t bits = (hi >= 32 ? ~0u : (hi <= 0 ? 0u : (1u << hi) - 1)) & (lo <= 0 ? ~0u : (lo >= 32 ? 0u : ~((1u << lo) - 1)));
#pragma unroll
              for (int j = 0; j < 32; j++) x[j] = bits >> j & 1 ? x[j] : 0xff800000u;      // -inf
            }
          };
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          auto maxima = [&](int ch, uint32_t* x) {
            hide(ch, x);
#pragma unroll
            for (int j = 0; j < 32; j += 2)
              mx[(j >> 1) & 3] = fmaxf(mx[(j >> 1) & 3], fmaxf(__uint_as_float(x[j]), __uint_as_float(x[j + 1])));
          };
#pragma unroll 1
          for (int ch = ch0; ch < ch1; ch++) {
            uint32_t x[32];
            tmem_ld_32x32b_x32(t_s + ch * 32, x);
            tmem_ld_wait();
            maxima(ch, x);
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
          auto exps = [&](int ch, uint32_t* x) {
            hide(ch, x);
            uint32_t pk[16];
#pragma unroll
            for (int j = 0; j < 16; j++) {
              const float p0 = sh_exp2(fmaf(__uint_as_float(x[2 * j]), sl2, nmb));
              const float p1 = sh_exp2(fmaf(__uint_as_float(x[2 * j + 1]), sl2, nmb));
              rs[(j & 1) * 2] += p0;
              rs[(j & 1) * 2 + 1] += p1;
              pk[j] = pack_bf16x2(p0, p1);       // the product takes bf16; the sum keeps 32 bits
            }
            tmem_st_32x32b_x16(t_s + ch * 16, pk);       // over columns that have been read
          };
#pragma unroll 1
          for (int ch = ch0; ch < ch1; ch++) {
            uint32_t x[32];
            tmem_ld_32x32b_x32(t_s + ch * 32, x);
            tmem_ld_wait();
            exps(ch, x);
          }
          l += (rs[0] + rs[1]) + (rs[2] + rs[3]);
          tmem_st_wait();
        }
        if ((c_lo & 15) || (c_hi & 15)) {        // rows of V beside the range that the product's steps of 16 keys reach
          if (nsel == 1 || off == 0) {
            const uint32_t st = gt % NV;
            if (!mbar_wait(&v_full[st], (gt / NV) & 1u, abort_word)) goto done;
            const int lo0 = c_lo & ~15, hi1 = (c_hi + 15) & ~15, nlo = c_lo - lo0, beside = nlo + hi1 - c_hi;
            for (int j = lane_row; j < beside * 8 * NH; j += 128) {
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
      // ---- the piece's rows: two slots up to 128 rows, one for each group of warps
      const long slot = (long)c.b.part_row + (long)(c.h + (int)blockIdx.x - c.b.seg0) * (nsel == 2 ? 1 : 2) * (c.b.ntok * G);
      const long at = slot + (nsel == 2 ? tok_first * G : (int)off * rows) + row;
      if (first < n) {
        if (row_valid) p.part_ml[at] = make_float2(l != l && m == -INFINITY ? 0.f : m * sl2, l);      // scores without a number count
        if (!mbar_wait(&o_full[w], oc & 1u, abort_word)) goto done;
        oc++;
        tc_fence_after();
        if (warp_valid) {
          float* dst = p.part_o + at * D;
#pragma unroll 1
          for (int ch = 0; ch < D / 32; ch++) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(t_o + w * 128 + ch * 32, r);
            tmem_ld_wait();
            if (row_valid) {
#pragma unroll
              for (int j = 0; j < 8; j++)
                reinterpret_cast<uint4*>(dst + ch * 32)[j] = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[w]);
      } else if (row_valid) {
        p.part_ml[at] = make_float2(-INFINITY, 0.f);     // a piece of one tile is the other group's: no rows of mine
      }
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

// Partial results of the prefix and of the sequence's own keys by their maxima and sums; WARPS warps a (token, head).
template <int D, int WARPS>
__global__ void __launch_bounds__(128) shared_join_kernel(const SharedParams p) {
  constexpr int V = D / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % WARPS;
  const long id = (long)blockIdx.x * (4 / WARPS) + warp / WARPS;
  const int t = (int)(id / p.Hq), hq = (int)(id - (long)t * p.Hq);
  const int* tok_base = p.plan + plan_tokens_at(p.blocks);
  int which[2] = {-1, -2};
  if (t < p.rows) which[0] = __ldg(tok_base + t), which[1] = __ldg(tok_base + p.tokens + t);
  const int h = hq / p.G, g = hq - h * p.G;
  long at[2];
  int n[2], pitch[2];
#pragma unroll
  for (int k = 0; k < 2; k++) {
    at[k] = n[k] = pitch[k] = 0;
    if (which[k] < 0) continue;
    const int2 head = __ldg(reinterpret_cast<const int2*>(p.plan + p.heads_at) + (long)which[k] * p.Hkv + h);
    const int2 tok = __ldg(reinterpret_cast<const int2*>(reinterpret_cast<const SharedBase*>(p.plan + p.bases_at) + which[k]));
    pitch[k] = tok.y * p.G;
    at[k] = (long)head.x + (t - tok.x) * p.G + g;
    n[k] = head.y;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");       // by every thread: what follows this kernel counts on those in front of it
  float acc[V], sum = 0.f, top = -INFINITY;
#pragma unroll
  for (int j = 0; j < V; j++) acc[j] = 0.f;
  const int all = n[0] + n[1];
  auto row_of = [&](int i) -> long { return i < n[0] ? at[0] + (long)i * pitch[0] : at[1] + (long)(i - n[0]) * pitch[1]; };
  for (int i0 = sub; i0 < all; i0 += 32 * WARPS) {         // a lane a partial result: maximum and sum
    const int mine = i0 + lane * WARPS, m = min(32, (all - i0 + WARPS - 1) / WARPS);
    const float2 e = lane < m ? p.part_ml[row_of(mine)] : make_float2(-INFINITY, 0.f);
    const float now = fmaxf(top, warp_reduce_max(e.x));
    if (now == -INFINITY) continue;
    const float old = sh_exp2(top - now);        // 0 in front of the first
    top = now;
    const float f = e.x > -INFINITY ? sh_exp2(e.x - now) : 0.f;
    sum = sum * old + warp_reduce_sum(e.x > -INFINITY ? f * e.y : 0.f);
#pragma unroll
    for (int j = 0; j < V; j++) acc[j] *= old;
#pragma unroll 4
    for (int i = 0; i < m; i++) {
      const float w = __shfl_sync(0xffffffffu, f, i);
      const float* o = p.part_o + row_of(i0 + i * WARPS) * D + lane * V;
      float x[V];
      if constexpr (V == 4) *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(o);
      else *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(o);
#pragma unroll
      for (int j = 0; j < V; j++) acc[j] += w == 0.f ? 0.f : w * x[j];       // where a group of warps had no tile, nothing was left
    }
  }
  if constexpr (WARPS == 4) {
    __shared__ float4 parts[3][33];
    if (sub > 0) {
      parts[sub - 1][lane] = make_float4(acc[0], acc[1], V == 4 ? acc[V - 2] : 0.f, V == 4 ? acc[V - 1] : 0.f);
      if (lane == 0) parts[sub - 1][32] = make_float4(top, sum, 0.f, 0.f);
    }
    __syncthreads();
    if (sub > 0) return;
#pragma unroll
    for (int k = 0; k < 3; k++) {
      const float4 e = parts[k][32], x = parts[k][lane];
      const float now = fmaxf(top, e.x);
      if (now == -INFINITY) continue;
      const float f = sh_exp2(top - now), fo = sh_exp2(e.x - now);
      top = now;
      sum = f * sum + fo * e.y;
      acc[0] = f * acc[0] + fo * x.x;
      acc[1] = f * acc[1] + fo * x.y;
      if constexpr (V == 4) acc[2] = f * acc[2] + fo * x.z, acc[3] = f * acc[3] + fo * x.w;
    }
  }
  if (which[1] == -2) return;                    // behind the last sequence: left as it is
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
  int block_size, max_blocks, Hq, Hkv, D, blocks, tokens, bases_at, max_bases;
};

// Maps of the queries (four boxes) or of a pair of caches (whole tiles and pieces), kept by what they encode.
struct SharedMapKey {
  const void* base[2];
  uint64_t dims[4], strides[3];
  uint32_t boxes[4];
  bool operator==(const SharedMapKey& o) const { return memcmp(this, &o, sizeof(*this)) == 0; }
};
struct SharedMapHash {
  size_t operator()(const SharedMapKey& k) const {
    const uint64_t* w = reinterpret_cast<const uint64_t*>(&k);
    uint64_t h = 0;
    for (size_t i = 0; i < sizeof(k) / 8; i++) h = (h ^ w[i]) * 0x9e3779b97f4a7c15ull, h ^= h >> 29;
    return (size_t)h;
  }
};
struct SharedMaps {
  CUtensorMap map[4];
};

// box i: 64 columns of all heads of a group by boxes[i] tokens, or of boxes[i] tokens of a page (keys and values in turn)
static int shared_maps(SharedMaps* out, const SharedMapKey& key, bool queries) {
  static std::unordered_map<SharedMapKey, SharedMaps, SharedMapHash> maps;
  static std::mutex mu;
  std::lock_guard<std::mutex> g(mu);
  auto it = maps.find(key);
  if (it == maps.end()) {
    SharedMaps m;
    for (int i = 0; i < 4; i++) {
      const uint32_t box[4] = {64, queries ? (uint32_t)key.dims[1] : 1u, queries ? 1u : key.boxes[i], queries ? key.boxes[i] : 1u};
      const int rc = make_tmap(&m.map[i], key.base[queries ? 0 : i & 1], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, key.dims, key.strides, box,
                               CU_TENSOR_MAP_SWIZZLE_128B);
      if (rc) return rc;
    }
    if (maps.size() > 2048) maps.clear();
    it = maps.emplace(key, m).first;
  }
  *out = it->second;
  return 0;
}

template <int D>
static int launch_shared(const SharedMaps& q, const SharedMaps& kv, const SharedParams& p, cudaStream_t stream) {
  const cudaError_t e = allow_smem<&attn_shared_kernel<D>>(SharedCfg<D>::SMEM);
  if (e != cudaSuccess) return (int)e;
  attn_shared_kernel<D><<<p.blocks, SH_THREADS, SharedCfg<D>::SMEM, stream>>>(q.map[0], q.map[1], q.map[2], q.map[3], kv.map[0],
                                                                                  kv.map[1], kv.map[2], kv.map[3], p);
  const int rc = B200_CHECK_LAUNCH();
  if (rc) return rc;
  // Few rows may have many partial results, up to two of each block: four warps a row.  They exchange theirs in shared memory that is not free beside
  // the attention's blocks, so they start behind those; blocks without begin early (192 sequences behind 2048 tokens 134 -> 131 us).
  const long rows = (long)p.rows * p.Hq;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows <= 4096 ? rows : (rows + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = rows <= 4096 ? 0 : 1;
  return (int)(rows <= 4096 ? cudaLaunchKernelEx(&cfg, shared_join_kernel<D, 4>, p) : cudaLaunchKernelEx(&cfg, shared_join_kernel<D, 1>, p));
}

}  // namespace b200

B200_API int b200_shared_plan(const b200::PlanArgs* args) {
  using namespace b200;
  const PlanArgs& a = *args;
  if (a.seqs < 0 || a.groups < 0 || a.tokens < 0 || a.G < 1 || a.G > 128 || a.Hkv < 1 || a.blocks < 1) return 9950;
  const int per = 2 * (128 / a.G);
  if ((long)a.max_bases < (long)a.groups + a.seqs + 2 * ((long)a.tokens / per) || (a.bases_at & 3) ||
      a.bases_at < plan_tokens_at(a.blocks) + 2 * a.tokens + a.groups || ((uintptr_t)a.plan & 15))
    return 9951;
  shared_plan_kernel<<<1, 1024, 0, a.stream>>>(a);
  return B200_CHECK_LAUNCH();
}

B200_API int b200_attn_shared(const b200::SharedArgs* args) {
  using namespace b200;
  const SharedArgs& a = *args;
  if (a.T <= 0 || a.tokens <= 0) return 0;
  const int bs = a.block_size;
  if (a.Hkv < 1 || a.Hq % a.Hkv || a.Hq / a.Hkv > 128 || (a.D != 64 && a.D != 128)) return 9955;
  if (bs < 8 || (bs < 128 && 128 % bs) || (bs > 128 && bs % 128)) return 9956;
  if ((a.q_stride & 7) || (a.out_stride & 7) || ((uintptr_t)a.q & 15) || ((uintptr_t)a.out & 15) || ((uintptr_t)a.k_cache & 15) ||
      ((uintptr_t)a.v_cache & 15) || (a.block_stride & 7) || (a.token_stride & 7) || (a.head_stride & 7))
    return 9957;
  const int G = a.Hq / a.Hkv, tpt = 128 / G;
  // what the pieces of a plan of these sizes have room for
  if (a.part_rows < 4L * a.tokens * a.Hq + (long)a.blocks * SH_ROWS) return 9958;
  const int rpl = bs < 128 ? bs : 128, piece = rpl < 32 ? rpl : 32;
  SharedMaps q, kv;
  SharedMapKey key;
  memset(&key, 0, sizeof(key));                // padding, if there is any, is compared
  key.base[0] = a.q;
  key.dims[0] = a.D, key.dims[1] = G, key.dims[2] = a.Hkv, key.dims[3] = a.T;
  key.strides[0] = a.D * 2, key.strides[1] = (uint64_t)G * a.D * 2, key.strides[2] = (uint64_t)a.q_stride * 2;
  key.boxes[0] = tpt, key.boxes[1] = G <= 64 ? 64 / G : 1, key.boxes[2] = tpt < 4 ? tpt : 4, key.boxes[3] = 1;
  int rc = shared_maps(&q, key, true);
  if (rc) return rc;
  key.base[0] = a.k_cache, key.base[1] = a.v_cache;
  key.dims[1] = a.Hkv, key.dims[2] = bs, key.dims[3] = a.num_blocks;
  key.strides[0] = (uint64_t)a.head_stride * 2, key.strides[1] = (uint64_t)a.token_stride * 2, key.strides[2] = (uint64_t)a.block_stride * 2;
  key.boxes[0] = key.boxes[1] = rpl, key.boxes[2] = key.boxes[3] = piece;
  rc = shared_maps(&kv, key, false);
  if (rc) return rc;
  SharedParams p;
  p.plan = a.plan;
  p.block_table = a.block_table;
  p.pitch = a.pitch;
  p.max_blocks = a.max_blocks;
  p.block_size = bs;
  p.page_shift = bs & (bs - 1) ? -1 : 31 - __builtin_clz(bs);
  p.rows_per_load = rpl;
  p.piece = piece;
  p.G = G; p.Hkv = a.Hkv; p.Hq = a.Hq; p.tpt = tpt;
  p.blocks = a.blocks;
  p.tokens = a.tokens;
  p.rows = (int)(a.T < a.tokens ? a.T : a.tokens);
  p.bases_at = a.bases_at;
  p.heads_at = plan_heads_at(a.bases_at, a.max_bases);
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.part_o = a.parts;
  p.part_ml = (float2*)(a.parts + a.part_rows * a.D);
  p.num_blocks_total = a.num_blocks;
  p.status = a.status;
  p.out = (__nv_bfloat16*)a.out;
  p.out_stride = a.out_stride;
  return a.D == 64 ? launch_shared<64>(q, kv, p, a.stream) : launch_shared<128>(q, kv, p, a.stream);
}
