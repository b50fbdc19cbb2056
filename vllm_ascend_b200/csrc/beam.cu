// Beam search on the device: the best continuations of a group of beams over the whole vocabulary, and beams' states brought
// behind their new parents.
//
//   total[g, w, v] = score[g, w] + logits[w, v] - log sum_v' exp(logits[w, v'])          the k best of each group, best first
//
// Selection reads the logits once.  A block walks a part of a row: every thread keeps a running maximum and the sum of exponentials
// under it; elements that reach the bound of the k-th best so far go to their warp's list in shared memory.  Within a row totals are
// ordered as logits are, so the lists need no sum.  The bound begins with the part's first elements, 32 a thread (16 of 32 bits): the k-th largest of the
// maxima of slices of them, which k elements or more reach, and not many more where values are in no order.  A warp whose list is full cuts it back to
// its k best, whose last raises the bound for all.  Keys carry the value and, below it, the place: no two are equal, ties go to the
// lowest place by themselves, and rows of equal values (masked ones) put nothing behind their first into a list.
// A second kernel, a block a group, adds up the sums of the parts, turns its beams' keys into totals and takes the best by their places in the lists.
// Threads' and parts' sums are joined in 64 bits and totals compared in 64: with thousands of candidates, sums of 32 bits would order near ones
// by their rounding.
// Many rows are bound by the instructions that are issued (three quarters of all places), half of them the walk: 768 rows of 151936 in bf16 take 85 us, 2.8
// TB/s; 730 of them that are read execute 82000 a row, 48000 in the walk, 16000 where elements reach the bound, the rest before and after.  Few rows are
// bound by what stands before and behind the walk, 3 and 4 us, and the second kernel, 5: 64 rows 22 us, 4 of 32000 13 us.
// Reordering: a thread owns 16 bytes of a row for all beams of a group and loads what they become before it stores the first.
#include "common.cuh"

namespace b200 {

constexpr int BEAM_THREADS = 512;
constexpr int BEAM_VEC = 8;                               // elements a thread takes of a tile
constexpr int BEAM_TILE = BEAM_THREADS * BEAM_VEC;
constexpr int BEAM_WARPS = BEAM_THREADS / 32;
constexpr int BEAM_MOST = 256;                            // k at most
constexpr int STAGE_BYTES = 64;                           // of a row on their way, a thread
constexpr int BEAM_ROOM = 1024;                           // candidates of a group that are looked at together
constexpr float kBeamLog2e = 1.4426950408889634f;

struct SelectArgs {
  const void* logits;
  const void* scores;            // [groups, width] of 32 or 64 bits
  uint64_t* keys;                // [rows, parts, k] best first
  int* counts;                   // [rows, parts]
  float* maxima;                 // [rows, parts]
  double* sums;                  // [rows, parts] of exp(x - maximum)
  void* out_scores;              // [groups, k] of as many
  int* out_parents;
  long* out_tokens;
  int* status;
  cudaStream_t stream;
  long row_stride;
  int groups, width, vocab, k, parts, per_part, fp32, wide;       // wide: scores of 64 bits
};

// ---------------------------------------------------------------- keys
// 32 bits that order floats as whole numbers, and back
__device__ __forceinline__ uint32_t order32(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);            // -0 and 0 are one value
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unorder32(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ uint64_t order64(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
  return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double unorder64(uint64_t k) {
  return __longlong_as_double((long long)(k & 0x8000000000000000ull ? k ^ 0x8000000000000000ull : ~k));
}

// a row's elements: value, then the lower place; 0 is no element
struct RowKey {
  uint64_t v;
  __device__ __forceinline__ bool above(const RowKey& o) const { return v > o.v; }
  __device__ __forceinline__ static RowKey none() { return {0ull}; }
  __device__ __forceinline__ RowKey other_lane(int o) const { return {__shfl_xor_sync(0xffffffffu, v, o)}; }
};
// a group's: total in 64 bits, then the lower place
struct GroupKey {
  uint64_t v;
  uint32_t place;                // complement of beam * vocab + token
  __device__ __forceinline__ bool above(const GroupKey& o) const { return v > o.v || (v == o.v && place > o.place); }
  __device__ __forceinline__ static GroupKey none() { return {0ull, 0u}; }
  __device__ __forceinline__ GroupKey other_lane(int o) const {
    return {__shfl_xor_sync(0xffffffffu, v, o), __shfl_xor_sync(0xffffffffu, place, o)};
  }
};

// ---------------------------------------------------------------- the k best of a list
// The k-th largest of one key a thread, found bit by bit (a barrier counts); all threads of the block.  Ranks by counting take as many steps as there are
// keys: 512 of them 20000 clocks, 64 bits 3000.
template <int LOW = 0>                                    // bits below LOW stay 0: a bound that more than k may reach
__device__ __forceinline__ RowKey kth_largest(RowKey mine, int k) {
  uint64_t last = 0;
#pragma unroll 1
  for (int bit = 63; bit >= LOW; bit--) {
    const uint64_t next = last | 1ull << bit;
    if (__syncthreads_count(mine.v >= next) >= k) last = next;
  }
  return {last};
}
template <int LOW = 0>
__device__ __forceinline__ GroupKey kth_largest(GroupKey mine, int k) {
  const uint64_t v = kth_largest<LOW>(RowKey{mine.v}, k).v;
  k -= __syncthreads_count(mine.v > v);                   // places decide among equal totals
  uint32_t last = 0;
#pragma unroll 1
  for (int bit = 31; bit >= 0; bit--) {
    const uint32_t next = last | 1u << bit;
    if (__syncthreads_count(mine.v == v && mine.place >= next) >= k) last = next;
  }
  return {v, last};
}

// The k-th largest of the maxima of slices of n elements, `top` that of a thread's (element i belongs to thread i mod 512); none where fewer than k
// slices have elements.  A slice is the lanes that leave 4 k of them, one at least.  Ends with a barrier.
template <typename Key, int... LOW>
__device__ __forceinline__ Key slice_bound(Key top, int n, int k, Key* slices, Key* bound) {
  const int tid = threadIdx.x;
  int lanes = 32;
  while (min(n, BEAM_THREADS) < 4 * k * lanes && lanes > 1) lanes >>= 1;
  const int count = (min(n, BEAM_THREADS) + lanes - 1) / lanes;
  if (count > 128) {
    for (int o = 1; o < lanes; o <<= 1) {
      const Key other = top.other_lane(o);
      if (other.above(top)) top = other;
    }
    return kth_largest<LOW...>(tid % lanes == 0 ? top : Key::none(), k);
  }
  for (int o = 1; o < lanes; o <<= 1) {
    const Key other = top.other_lane(o);
    if (other.above(top)) top = other;
  }
  if (tid % lanes == 0) slices[tid / lanes] = top;
  if (tid == 0) *bound = Key::none();
  __syncthreads();
  int rank = 0;                                           // all lanes of a slice count
#pragma unroll 4
  for (int j = tid % lanes; j < count; j += lanes) rank += slices[j].above(top);
  for (int o = 1; o < lanes; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
  if (tid % lanes == 0 && rank == k - 1) *bound = top;    // one slice, but for those without an element, all of them none
  __syncthreads();
  return *bound;
}

// The k best of n keys, best first, into keys[0..k); returns how many.  All threads of the block, the keys written before a barrier; `other` has
// room for half of the keys, 256 at least.  Ends with a barrier.  Loops stay rolled here and in the group's kernel: code that runs once takes as long as it
// is fetched from memory.
template <typename Key>
__device__ int select_best(Key* keys, Key* other, int n, int k, Key* slices, Key* bound, int* count) {
  const int tid = threadIdx.x;
  Key* from = keys;
  // Only k slices reach the bound: a quarter of the elements at most, or where a slice is a thread, its k elements for every 512; values in no order
  // take one pass.  128 are ranked sooner than thinned out (64 rows of 151936: 22 us, 25 with a pass from 64 on).
  for (bool more = n > max(2 * k, 128); more; more = n > max(3 * k, 256)) {
    Key top = Key::none();
#pragma unroll 1
    for (int i = tid; i < n; i += BEAM_THREADS)
      if (from[i].above(top)) top = from[i];
    if (tid == 0) *count = 0;
    const Key least = slice_bound(top, n, k, slices, bound);
#pragma unroll 1
    for (int i = tid; i < n; i += BEAM_THREADS) {
      const Key key = from[i];
      if (!least.above(key)) other[atomicAdd(count, 1)] = key;
    }
    __syncthreads();
    n = *count;
    Key* swap = from;
    from = other;
    other = swap;
    __syncthreads();
  }
  if (n > k && n > 128 && n <= BEAM_THREADS) {            // down to k, which are ranked sooner
    const Key own = tid < n ? from[tid] : Key::none();
    const Key least = kth_largest(own, k);
    if (tid == 0) *count = 0;
    __syncthreads();
    if (tid < n && !least.above(own)) from[atomicAdd(count, 1)] = own;
    __syncthreads();
    n = *count;
    __syncthreads();
  }
  // ranked by counting: 3 k elements at most, the block's threads shared between them
  static_assert(3 * BEAM_MOST <= 2 * BEAM_THREADS, "two elements a thread");
  int each = 1;
  while (each < 32 && n * each * 2 <= BEAM_THREADS) each <<= 1;
  Key own[2];
  int rank[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int at = i * BEAM_THREADS + tid / each;         // a second one only where each is 1
    own[i] = at < n && (i == 0 || each == 1) ? from[at] : Key::none();
    rank[i] = 0;
    if (own[i].above(Key::none())) {
#pragma unroll 4
      for (int j = tid % each; j < n; j += each) rank[i] += from[j].above(own[i]);
    }
    if (i == 0)
      for (int o = 1; o < each; o <<= 1) rank[i] += __shfl_xor_sync(0xffffffffu, rank[i], o);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; i++)
    if (tid % each == 0 && own[i].above(Key::none()) && rank[i] < k) keys[rank[i]] = own[i];
  __syncthreads();
  return min(n, k);
}

// ---------------------------------------------------------------- exponentials and logarithms in 64 bits
// e^x for x <= 0 and log x for x >= 1 in 64 bits, by their series: short loops where the library's functions are a few hundred instructions that a
// kernel of this length waits for.
__constant__ double kInverseOdd[16] = {1., 1. / 3, 1. / 5, 1. / 7, 1. / 9, 1. / 11, 1. / 13, 1. / 15, 1. / 17, 1. / 19, 1. / 21, 1. / 23,
                                           1. / 25, 1. / 27, 1. / 29, 1. / 31};
__constant__ double kInverseFactorial[14] = {1., 1., 1. / 2, 1. / 6, 1. / 24, 1. / 120, 1. / 720, 1. / 5040, 1. / 40320, 1. / 362880, 1. / 3628800,
                                             1. / 39916800, 1. / 479001600, 1. / 6227020800.};
template <int TERMS = 13>
__device__ __forceinline__ double series_exp(double x) {       // e^x = 2^n e^r, |r| <= log(2) / 2; to r^(TERMS + 1) / (TERMS + 1)!
  if (x < -700.) return 0.;
  const double n = rint(x * 1.4426950408889634), r = x - n * 0.69314718055994531;
  double e = kInverseFactorial[TERMS];
#pragma unroll 1
  for (int i = TERMS - 1; i >= 0; i--) e = e * r + kInverseFactorial[i];
  return e * __longlong_as_double((long long)(1023 + (int)n) << 52);
}
__device__ __forceinline__ double series_log(double x) {       // log 2^n m = n log 2 + 2 atanh((m - 1) / (m + 1)), m in [0.75, 1.5)
  const uint64_t b = (uint64_t)__double_as_longlong(x);
  int n = (int)(b >> 52) - 1023;
  double m = __longlong_as_double((long long)((b & 0xfffffffffffffull) | 0x3ff0000000000000ull));
  if (m >= 1.5) m *= 0.5, n++;
  const double d = m + 1.;
  double inv = (double)(1.f / (float)d);
  inv = inv * (2. - d * inv);
  inv = inv * (2. - d * inv);
  const double z = (m - 1.) * inv, q = z * z;                  // |z| <= 0.2: sixteen terms are 3e-24
  double t = 0.;
#pragma unroll 1
  for (int i = 15; i >= 0; i--) t = t * q + kInverseOdd[i];
  return n * 0.69314718055994531 + 2. * z * t;
}

// ---------------------------------------------------------------- parts of rows
__device__ __forceinline__ float beam_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Eight elements on their way to a place in shared memory that belongs to the thread: those of the row in [0, end), -inf beside.
template <typename T>
__device__ __forceinline__ void bring(T* to, const T* row, int at, int end) {
  if (at >= 0 && at + BEAM_VEC <= end) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to) + 16 * i), "l"(reinterpret_cast<const uint4*>(row + at) + i)
                   : "memory");
  } else {
#pragma unroll 1
    for (int j = 0; j < BEAM_VEC; j++) to[j] = at + j >= 0 && at + j < end ? row[at + j] : T(-INFINITY);
  }
}
// Eight elements and the largest of them; of 16 bits two are compared at a time.
template <typename T>
__device__ __forceinline__ float take(const T* from, float* x) {
  const uint4 a = *reinterpret_cast<const uint4*>(from);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
  if constexpr (sizeof(T) == 2) {
    auto pair = [&](int i) { return *reinterpret_cast<const __nv_bfloat162*>(w + i); };
    const float2 top = __bfloat1622float2(__hmax2(__hmax2(pair(0), pair(1)), __hmax2(pair(2), pair(3))));
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    return fmaxf(top.x, top.y);
  } else {
    const uint4 b = *(reinterpret_cast<const uint4*>(from) + 1);
    const uint32_t v[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = __uint_as_float(w[i]), x[4 + i] = __uint_as_float(v[i]);
    float top = x[0];
#pragma unroll
    for (int i = 1; i < BEAM_VEC; i++) top = fmaxf(top, x[i]);
    return top;
  }
}

// two sums or products of 32 bits at a time
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 y;
  asm("{\n.reg .b64 p, q;\nmov.b64 p, {%2, %3};\nmov.b64 q, {%4, %5};\nadd.rn.f32x2 p, p, q;\nmov.b64 {%0, %1}, p;\n}"
      : "=f"(y.x), "=f"(y.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return y;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 y;
  asm("{\n.reg .b64 p, q;\nmov.b64 p, {%2, %3};\nmov.b64 q, {%4, %5};\nmul.rn.f32x2 p, p, q;\nmov.b64 {%0, %1}, p;\n}"
      : "=f"(y.x), "=f"(y.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return y;
}

__device__ __forceinline__ double score_of(const SelectArgs& a, long row) {
  return a.wide ? ((const double*)a.scores)[row] : (double)((const float*)a.scores)[row];
}
__device__ __forceinline__ bool is_score(double s) { return s > -INFINITY && s < INFINITY; }

// A warp's list: room for k keys and more, and for what a vector of its lanes may add.
__host__ __device__ constexpr int list_room(int k) { return (k + 31) / 32 * 32 + 32 + 32 * BEAM_VEC; }
constexpr int LIST_MOST = list_room(BEAM_MOST) / 32;
static_assert(BEAM_MOST * BEAM_WARPS * 8 <= BEAM_THREADS * STAGE_BYTES, "the warps' best lie in the place of the elements");
static_assert(BEAM_WARPS * list_room(1) >= BEAM_THREADS + BEAM_MOST * BEAM_WARPS / 2, "slices and half of the keys lie in the place of the lists");
// keys that are looked at together in the end: the warps' k best at least
__host__ __device__ constexpr int list_all(int k) { return BEAM_WARPS * k > 1024 ? BEAM_WARPS * k : 1024; }

// A warp's n > k different keys cut back to its k best, in no order; returns the last of them, found bit by bit.
__device__ __noinline__ uint64_t cut_back(uint64_t* list, int n, int k) {
  const int lane = threadIdx.x & 31;
  uint64_t own[LIST_MOST];
  __syncwarp();
#pragma unroll
  for (int i = 0; i < LIST_MOST; i++) own[i] = i * 32 + lane < n ? list[i * 32 + lane] : 0;
  // bits above the highest in which two keys differ are those of all
  const uint64_t some = __shfl_sync(0xffffffffu, own[0], 0);
  uint64_t differ = 0;
#pragma unroll
  for (int i = 0; i < LIST_MOST; i++) differ |= own[i] ? own[i] ^ some : 0;
  const uint32_t high = __reduce_or_sync(0xffffffffu, (uint32_t)(differ >> 32)), low = __reduce_or_sync(0xffffffffu, (uint32_t)differ);
  const int first = high ? 63 - __clz(high) : 31 - __clz(low | 1);
  uint64_t last = some & ~((2ull << first) - 1);
  for (int bit = first; bit >= 0; bit--) {
    const uint64_t next = last | 1ull << bit;
    int reach = 0;
#pragma unroll
    for (int i = 0; i < LIST_MOST; i++) reach += own[i] >= next;
    reach = __reduce_add_sync(0xffffffffu, reach);
    if (reach >= k) last = next;
    if (reach == k) break;
  }
  __syncwarp();
  int at = 0;
#pragma unroll
  for (int i = 0; i < LIST_MOST; i++) {
    const uint32_t who = __ballot_sync(0xffffffffu, own[i] >= last);
    if (own[i] >= last) list[at + __popc(who & ((1u << lane) - 1))] = own[i];
    at += __popc(who);
  }
  __syncwarp();
  return last;
}

template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS, 2) select_rows_kernel(const SelectArgs a) {
  extern __shared__ __align__(16) uint8_t beam_smem[];
  __shared__ RowKey first_bound;
  __shared__ unsigned long long bound;             // what a key has to reach, the k-th best of some that were seen
  __shared__ int held[BEAM_WARPS], count;          // keys in the warps' lists
  __shared__ float warp_max[BEAM_WARPS];
  __shared__ double warp_sum[BEAM_WARPS];
  const int row = blockIdx.x / a.parts, part = blockIdx.x % a.parts, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // once all blocks run, groups' may take their places and wait
  if (!is_score(score_of(a, row))) return;            // the beam has ended: the second kernel asks its score first
  const T* x0 = (const T*)a.logits + (long)row * a.row_stride;
  // vectors lie on 16-byte boundaries of memory, whatever the row's first element does; a vector holds elements [at, at + 8)
  const int shift = (int)(((uintptr_t)x0 & 15) / sizeof(T));
  const int from = part * a.per_part - shift, to = (int)min((long)from + a.per_part, (long)a.vocab);
  const int room = list_room(a.k);
  constexpr int STAGES = STAGE_BYTES / (BEAM_VEC * (int)sizeof(T));
  T* stage = reinterpret_cast<T*>(beam_smem) + tid * BEAM_VEC;       // [stages][threads][8], a thread's own
  uint64_t* lists = reinterpret_cast<uint64_t*>(beam_smem + BEAM_THREADS * STAGE_BYTES);
  uint64_t* list = lists + warp * room;
  RowKey* slices = reinterpret_cast<RowKey*>(lists);       // while there are no lists, and when they have been read
  // Of the elements at -inf only the row's first ones can be wanted: where fewer than k others are, k of them lie in the first 2 k places.
  auto key_of = [&](float x, int at) -> uint64_t {
    return at >= 0 && at < to && (x > -INFINITY || at < 2 * a.k) ? ((uint64_t)order32(x) << 32) | (uint32_t)~at : 0;
  };
  // ---- the bound that the first elements give, 32 a thread (16 of fp32)
  const int at0 = from + tid * BEAM_VEC;
#pragma unroll 1
  for (int i = 0; i < STAGES; i++) {
    bring(stage + i * BEAM_TILE, x0, at0 + i * BEAM_TILE < to ? at0 + i * BEAM_TILE : a.vocab, a.vocab);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  float high = -INFINITY;
#pragma unroll
  for (int i = 0; i < STAGES; i++) {
    float x[BEAM_VEC];
    const float t = take(stage + i * BEAM_TILE, x);
    if (at0 + i * BEAM_TILE < to) high = fmaxf(high, t);
  }
  // told apart by their threads; of the bound the value counts, all that equal it reach it
  const RowKey top = slice_bound<RowKey, 32>(RowKey{high > -INFINITY ? ((uint64_t)order32(high) << 32) | (uint32_t)~tid : 0ull}, BEAM_THREADS, a.k, slices, &first_bound);
  if (tid == 0) bound = top.v >> 32 << 32;
  if (lane == 0) held[warp] = 0;
  __syncthreads();
  // ---- all of the part, a warp by itself
  float m = -INFINITY, s = 0.f, reach = 0.f;
  uint64_t least = 0;
  int place = 0;
#pragma unroll 1
  for (int at = at0; at - tid * BEAM_VEC < to; at += STAGES * BEAM_TILE) {
#pragma unroll
    for (int st = 0; st < STAGES; st++) {
      const int mine = at + st * BEAM_TILE;
      if (mine - tid * BEAM_VEC >= to) break;
      if (st == 0) {                                 // the bound, as others have raised it
        least = *(volatile unsigned long long*)&bound;
        reach = least ? unorder32((uint32_t)(least >> 32)) : -INFINITY;
        // equal values count up to there
        place = reach == -INFINITY ? 2 * a.k - 1 : ((uint32_t)least ? (int)~(uint32_t)least : a.vocab);
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      float x[BEAM_VEC];
      const float t = take(stage + st * BEAM_TILE, x);
      // No branches: with a warp's 32 maxima, one of them rises in most steps.  The kernel is bound by its instructions, about 80 a vector.
      const bool live = mine < to;
      const float now = live ? fmaxf(m, t) : m;
      // differences from the maximum are taken before the factor: a product of the maximum would carry its rounding into every term
      const float under = now == -INFINITY ? 0.f : now;
      float2 u[2];
#pragma unroll
      for (int j = 0; j < BEAM_VEC; j += 2) {
        const float2 d = mul2(add2(make_float2(x[j], x[j + 1]), make_float2(-under, -under)), make_float2(kBeamLog2e, kBeamLog2e));
        const float2 e = make_float2(beam_exp2(d.x), beam_exp2(d.y));          // a NaN or +inf: NaN
        u[j >> 1 & 1] = j < 4 ? e : add2(u[j >> 1 & 1], e);
      }
      u[0] = add2(u[0], u[1]);
      const float all = fmaf(s, beam_exp2(fminf(m - under, 0.f) * kBeamLog2e), u[0].x + u[0].y);       // s is 0 under -inf
      s = live ? all : s;
      m = now;
      const bool hit = live & (t >= reach) & ((t > reach) | (mine <= place));
      if (__any_sync(0xffffffffu, hit)) {
        if (hit) {
          uint32_t which = 0;
#pragma unroll
          for (int j = 0; j < BEAM_VEC; j++) which |= x[j] >= reach ? 1u << j : 0u;
          while (which) {
            const int j = __ffs(which) - 1;
            which &= which - 1;
            const uint64_t key = key_of((float)stage[st * BEAM_TILE + j], mine + j);
            if (key != 0 && key >= least) list[atomicAdd(&held[warp], 1)] = key;
          }
        }
        __syncwarp();
        const int n = *(volatile int*)&held[warp];
        if (n > room - 32 * BEAM_VEC) {              // the next vector has room
          const uint64_t last = cut_back(list, n, a.k);
          if (lane == 0) {
            held[warp] = a.k;
            atomicMax(&bound, (unsigned long long)last);
          }
        }
        __syncwarp();
      }
      const int next = mine + STAGES * BEAM_TILE;
      if (next < to) bring(stage + st * BEAM_TILE, x0, next, a.vocab);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  }
  // ---- the block's k best, in the place of the elements
  asm volatile("cp.async.wait_all;" ::: "memory");
  uint64_t* all = reinterpret_cast<uint64_t*>(beam_smem);
  {
    __syncthreads();
    int n = 0;
    for (int i = 0; i < BEAM_WARPS; i++) n += held[i];
    const bool many = n > list_all(a.k);           // values in an order against the bound
    n = held[warp];
    if (many && n > a.k) {
      const uint64_t last = cut_back(list, n, a.k);
      if (lane == 0) atomicMax(&bound, (unsigned long long)last);
      n = a.k;
    }
    if (tid == 0) count = 0;
    __syncthreads();
    const uint64_t least = bound;
#pragma unroll 1
    for (int i = lane; i < n; i += 32)
      if (list[i] >= least) all[atomicAdd(&count, 1)] = list[i];
    __syncthreads();
  }
  const int found = count;
  __syncthreads();
  RowKey* best = reinterpret_cast<RowKey*>(all);
  const int got = select_best<RowKey>(best, slices + BEAM_THREADS, found, a.k, slices, &first_bound, &count);
  const long slot = (long)row * a.parts + part;
  for (int i = tid; i < got; i += BEAM_THREADS) a.keys[slot * a.k + i] = all[i];
  // ---- the part's maximum and its sum under it
  high = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
  if (lane == 0) warp_max[warp] = high;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < BEAM_WARPS; i++) high = fmaxf(high, warp_max[i]);
  // in 64 bits: where one element stands above a flat row, all threads have the same distance, and its rounding would not average out (3e-7);
  // eight terms are off by 2e-10
  double sum = m == -INFINITY ? (double)s : (double)s * series_exp<8>((double)m - (double)high);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) warp_sum[warp] = sum;
  __syncthreads();
  if (tid < 32) {
    sum = lane < BEAM_WARPS ? warp_sum[lane] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if (tid == 0) {
    a.maxima[slot] = high;
    a.sums[slot] = sum;
    a.counts[slot] = got;
  }
}

// ---------------------------------------------------------------- groups
struct GroupList {
  GroupKey keys[BEAM_ROOM + BEAM_MOST], other[(BEAM_ROOM + BEAM_MOST) / 2 + 128];
  GroupKey slices[BEAM_THREADS];
  GroupKey bound;
  int count;
};

__global__ void __launch_bounds__(BEAM_THREADS, 1) select_groups_kernel(const SelectArgs a) {
  extern __shared__ __align__(16) uint8_t beam_smem[];
  GroupList& list = *reinterpret_cast<GroupList*>(beam_smem);
  double* norm = reinterpret_cast<double*>(beam_smem + sizeof(GroupList));      // log of a beam's sum; NaN: it has no candidates
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");       // the blocks of rows have ended, and what came in front of them
  for (int w = tid >> 5; w < a.width; w += BEAM_WARPS) {          // a warp a beam, a lane a part
    const long row = (long)g * a.width + w;
    double l = __longlong_as_double(0x7ff8000000000000ll);
    if (is_score(score_of(a, row))) {
      float top = -INFINITY;
      for (int p = lane; p < a.parts; p += 32) top = fmaxf(top, a.maxima[row * a.parts + p]);
      top = warp_reduce_max(top);
      double sum = 0.0;
      for (int p = lane; p < a.parts; p += 32) {
        const float mp = a.maxima[row * a.parts + p];
        const double sp = a.sums[row * a.parts + p];
        sum += mp == -INFINITY ? sp : sp * series_exp((double)mp - (double)top);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (top > -INFINITY && top < INFINITY && sum >= 1.0 && sum < 1e300) l = (double)top + series_log(sum);      // the largest adds 1; NaN fails all
    }
    if (lane == 0) norm[w] = l;
  }
  __syncthreads();
  // Candidates by their places in the lists, which are sorted: the best of all lists come first, few behind them reach what those leave, and where no
  // list has one that does, none comes behind it.  A beam without a distribution offers its first tokens at -inf.
  const int lists = a.width * a.parts, levels = max(1, BEAM_ROOM / lists);
  GroupKey least = GroupKey::none();
  int n = 0;
  for (int c0 = 0; c0 < a.k; c0 += levels) {
    if (tid == 0) list.count = n;
    __syncthreads();
    bool any = false;
#pragma unroll 1
    for (int i = tid; i < min(levels, a.k - c0) * lists; i += BEAM_THREADS) {
      const int c = c0 + i / lists, j = i % lists, w = j / a.parts, p = j - w * a.parts;
      const long row = (long)g * a.width + w, slot = row * a.parts + p;
      const double l = norm[w];
      GroupKey key = GroupKey::none();
      if (l != l) {
        if (p == 0 && c < a.vocab) key = {order64(-INFINITY), ~(uint32_t)(w * a.vocab + c)};
      } else if (c < a.counts[slot]) {
        const uint64_t r = a.keys[slot * a.k + c];
        const float x = unorder32((uint32_t)(r >> 32));
        key = {order64(score_of(a, row) + ((double)x - l)), ~((uint32_t)(w * a.vocab) + ~(uint32_t)r)};
      }
      if (key.above(least)) {
        list.keys[atomicAdd(&list.count, 1)] = key;
        any = true;
      }
    }
    any = __syncthreads_or(any);
    n = list.count;
    __syncthreads();
    if (!any) break;
    n = select_best<GroupKey>(list.keys, list.other, n, a.k, list.slices, &list.bound, &list.count);
    if (n == a.k) least = list.keys[a.k - 1];
    __syncthreads();
  }
  for (int i = tid; i < a.k; i += BEAM_THREADS) {
    const GroupKey key = list.keys[i];
    const uint32_t place = ~key.place;
    const long to = (long)g * a.k + i;
    const double total = unorder64(key.v);
    if (a.wide) ((double*)a.out_scores)[to] = total;
    else ((float*)a.out_scores)[to] = (float)total;
    a.out_parents[to] = (int)(place / (uint32_t)a.vocab);
    a.out_tokens[to] = (long)(place % (uint32_t)a.vocab);
  }
}

// ---------------------------------------------------------------- states behind their new parents
// One tensor whose rows follow the beams: row r is `outer` runs of bytes, `outer_stride` apart, each of `units` units of
// `unit_bytes`; a unit holds `unit_tokens` tokens (0: the row is copied whole).
struct BeamTensor {
  uint8_t* base;
  long row_stride, outer_stride, unit_bytes, rows;
  int outer, units, unit_tokens, width;      // width: bytes that a thread moves at once
};

struct ReorderArgs {
  const BeamTensor* tensors;
  const int* rows;               // [groups, beams] row of each beam, -1: no such beam
  const int* parents;            // [groups, beams] the beam of its group that it follows, -1: none
  const int* lengths;            // [groups] filled tokens of the beams' pages, or null
  int* status;
  cudaStream_t stream;
  int num_tensors, groups, beams, wide, sms;     // wide: the first so many tensors move 16 bytes at once
};

template <int BYTES>
struct Bits;
template <> struct Bits<16> { using type = uint4; };
template <> struct Bits<8> { using type = uint2; };
template <> struct Bits<4> { using type = uint32_t; };
template <> struct Bits<2> { using type = uint16_t; };
template <> struct Bits<1> { using type = uint8_t; };

constexpr int REORDER_BEAMS = 1024;        // beams of a group at most

// What rows become: from[w] for beam w's, -1: it stays; all blocks of a group find the same.  False where nothing moves.
__device__ __forceinline__ bool find_sources(const ReorderArgs& a, const BeamTensor& t, int* from, int* to) {
  bool any = false;
  for (int w = threadIdx.x; w < a.beams; w += blockDim.x) {
    const long b = (long)blockIdx.z * a.beams;
    const int row = a.rows[b + w], p = a.parents[b + w];
    int source = -1;
    bool bad = row < -1 || row >= t.rows || p < -1 || p >= a.beams;
    if (!bad && row >= 0 && p >= 0 && p != w) {
      source = a.rows[b + p];
      bad = source < 0 || source >= t.rows;
      if (source == row) source = -1;
    }
    if (bad) {
      source = -1;
      atomicExch(a.status, B200_BAD_INDEX);
    }
    from[w] = source;
    to[w] = row;
    any |= source >= 0;
  }
  return __syncthreads_or(any);
}

// bytes of a run that move
__device__ __forceinline__ long run_bytes(const ReorderArgs& a, const BeamTensor& t) {
  int units = t.units;
  if (t.unit_tokens > 0 && a.lengths) units = min((long)units, ((long)max(0, a.lengths[blockIdx.z]) + t.unit_tokens - 1) / t.unit_tokens);
  return (long)units * t.unit_bytes;
}

// A block's share of the positions in a row, `width` bytes each: `move` is called with the offset of each.
template <typename Move>
__device__ __forceinline__ void walk_row(const BeamTensor& t, long run, int width, Move move) {
  const long all = run * t.outer, step = (long)gridDim.x * blockDim.x * width;
  for (long at = ((long)blockIdx.x * blockDim.x + threadIdx.x) * width; at < all; at += step) {
    const long o = t.outer == 1 ? 0 : (all <= 0xffffffffl ? (long)((uint32_t)at / (uint32_t)run) : at / run);
    move(at + o * (t.outer_stride - run));
  }
}

// Up to MOST beams: what a thread's 16 bytes of all rows become is loaded before the first is stored.  Blocks walk several positions, so that what it
// takes to find the sources (three loads one behind the other) shows once: 64 rows of 2.1 MB in 4 layers 113 us (what moves, read and written, at 6.1 TB/s,
// 0.92 of a copy), 174 with one position a thread.  128 pages of 16 groups in 12 layers 41 us (0.85), 4 pages in 36 layers 15.
template <int MOST>
__global__ void __launch_bounds__(256, MOST == 16 ? 2 : 4) reorder_kernel(const ReorderArgs a) {
  __shared__ int from[MOST], to[MOST];
  const BeamTensor t = a.tensors[blockIdx.y];
  const long run = run_bytes(a, t);
  if (!find_sources(a, t, from, to) || run == 0) return;
  walk_row(t, run, 16, [&](long offset) {
    uint8_t* at = t.base + offset;
    uint4 v[MOST];
#pragma unroll
    for (int w = 0; w < MOST; w++)
      if (w < a.beams && from[w] >= 0) v[w] = *reinterpret_cast<const uint4*>(at + (long)from[w] * t.row_stride);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int w = 0; w < MOST; w++)
      if (w < a.beams && from[w] >= 0) *reinterpret_cast<uint4*>(at + (long)to[w] * t.row_stride) = v[w];
  });
}

// Any number of beams and any alignment: a thread's loads go to its column of shared memory (asynchronously where 16 bytes move at once).
template <int BYTES>
__device__ __forceinline__ void move_staged(const BeamTensor& t, const int* from, const int* to, int beams, long offset, uint8_t* stage) {
  using V = typename Bits<BYTES>::type;
  uint8_t* at = t.base + offset;
  V* mine = reinterpret_cast<V*>(stage) + threadIdx.x;
  const int pitch = blockDim.x;
  for (int w = 0; w < beams; w++) {
    if (from[w] < 0) continue;
    const uint8_t* src = at + (long)from[w] * t.row_stride;
    if constexpr (BYTES == 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(mine + w * pitch)), "l"(src) : "memory");
    else
      mine[w * pitch] = *reinterpret_cast<const V*>(src);
  }
  if constexpr (BYTES == 16) asm volatile("cp.async.wait_all;" ::: "memory");
  for (int w = 0; w < beams; w++)
    if (from[w] >= 0) *reinterpret_cast<V*>(at + (long)to[w] * t.row_stride) = mine[w * pitch];
}

__global__ void __launch_bounds__(256) reorder_staged_kernel(const ReorderArgs a) {
  extern __shared__ __align__(16) uint8_t beam_smem[];
  int* from = reinterpret_cast<int*>(beam_smem);
  int* to = from + a.beams;
  uint8_t* stage = beam_smem + ((2 * a.beams * sizeof(int) + 15) & ~(size_t)15);
  const BeamTensor t = a.tensors[blockIdx.y];
  const long run = run_bytes(a, t);
  if (!find_sources(a, t, from, to) || run == 0) return;
  walk_row(t, run, t.width, [&](long offset) {
    switch (t.width) {
      case 16: move_staged<16>(t, from, to, a.beams, offset, stage); break;
      case 8: move_staged<8>(t, from, to, a.beams, offset, stage); break;
      case 4: move_staged<4>(t, from, to, a.beams, offset, stage); break;
      case 2: move_staged<2>(t, from, to, a.beams, offset, stage); break;
      default: move_staged<1>(t, from, to, a.beams, offset, stage); break;
    }
  });
}

}  // namespace b200

// ---------------------------------------------------------------- host
B200_API int b200_beam_select(const b200::SelectArgs* args) {
  using namespace b200;
  const SelectArgs& a = *args;
  if (a.groups <= 0) return 0;
  const long rows = (long)a.groups * a.width;
  if (a.width < 1 || a.vocab < 1 || a.k < 1 || a.k > BEAM_MOST || (long)a.k > (long)a.width * a.vocab) return 9930;
  if ((long)a.width * a.vocab > 0x7fffffffL || rows * a.parts > 0x7fffffffL || (long)a.width * a.parts * a.k > 0x7fffffffL) return 9931;
  // a walk counts up to eight tiles past a row's end
  if (a.vocab > 0x7fffffff - 8 * BEAM_TILE || a.parts < 1 || a.per_part < BEAM_VEC || a.per_part % BEAM_VEC ||
      (long)(a.parts - 1) * a.per_part >= (long)a.vocab + BEAM_VEC - 1 || (long)a.parts * a.per_part < (long)a.vocab + BEAM_VEC - 1)
    return 9932;
  const int row_smem = BEAM_THREADS * STAGE_BYTES + BEAM_WARPS * list_room(a.k) * 8, group_smem = (int)sizeof(GroupList) + a.width * 8;
  if ((long)a.width * a.parts > BEAM_ROOM) return 9933;      // a level of all lists is looked at together
  const unsigned grid = (unsigned)(rows * a.parts);
  cudaError_t e = a.fp32 ? allow_smem<&select_rows_kernel<float>>(112 * 1024) : allow_smem<&select_rows_kernel<__nv_bfloat16>>(112 * 1024);
  if (e == cudaSuccess) e = allow_smem<&select_groups_kernel>(64 * 1024);
  if (e != cudaSuccess) return (int)e;
  if (a.fp32) select_rows_kernel<float><<<grid, BEAM_THREADS, row_smem, a.stream>>>(a);
  else select_rows_kernel<__nv_bfloat16><<<grid, BEAM_THREADS, row_smem, a.stream>>>(a);
  int rc = B200_CHECK_LAUNCH();
  if (rc) return rc;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.groups);
  cfg.blockDim = dim3(BEAM_THREADS);
  cfg.dynamicSmemBytes = group_smem;
  cfg.stream = a.stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, select_groups_kernel, a);
}

B200_API int b200_beam_reorder(const b200::ReorderArgs* args) {
  using namespace b200;
  ReorderArgs a = *args;
  if (a.groups <= 0 || a.beams <= 0 || a.num_tensors <= 0) return 0;
  if (a.beams > REORDER_BEAMS || a.groups > 65535 || a.num_tensors > 65535 || a.wide < 0 || a.wide > a.num_tensors) return 9940;
  const int wide = a.beams <= 16 ? a.wide : 0, rest = a.num_tensors - wide;
  // blocks enough to fill the GPU a few times over, whatever the tensors' and the groups' number
  if (wide > 0) {
    const long pairs = (long)wide * a.groups;
    const dim3 grid((unsigned)((32L * a.sms + pairs - 1) / pairs), (unsigned)wide, (unsigned)a.groups);
    if (a.beams <= 4) reorder_kernel<4><<<grid, 256, 0, a.stream>>>(a);
    else if (a.beams <= 8) reorder_kernel<8><<<grid, 256, 0, a.stream>>>(a);
    else reorder_kernel<16><<<grid, 256, 0, a.stream>>>(a);
    const int rc = B200_CHECK_LAUNCH();
    if (rc) return rc;
  }
  if (rest > 0) {
    // a block's columns stay within 64 KB
    int threads = 256;
    while (threads * a.beams > 4096 && threads > 4) threads >>= 1;
    const int smem = ((2 * a.beams * 4 + 15) & ~15) + a.beams * threads * 16;
    const cudaError_t e = allow_smem<&reorder_staged_kernel>(80 * 1024);
    if (e != cudaSuccess) return (int)e;
    a.tensors += wide;
    const long pairs = (long)rest * a.groups, blocks = 32L * a.sms * (256 / threads);
    const dim3 grid((unsigned)((blocks + pairs - 1) / pairs), (unsigned)rest, (unsigned)a.groups);
    reorder_staged_kernel<<<grid, threads, smem, a.stream>>>(a);
  }
  return B200_CHECK_LAUNCH();
}
