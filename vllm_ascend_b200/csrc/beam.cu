// Beam search on the device: the best continuations of a group of beams over the whole vocabulary, and beams' states brought
// behind their new parents.
//
//   total[g, w, v] = score[g, w] + logits[w, v] - log sum_v' exp(logits[w, v'])          the k best of each group, best first
//
// Selection reads the logits once.  A block walks a part of a row: every thread keeps a running maximum and the sum of exponentials
// under it, and puts elements above the part's k-th best so far into a list in shared memory; within a row totals are ordered as
// logits are, so the list needs no sum.  A list that grows is cut back to its k best: the k-th largest of the maxima of at least 2 k
// slices of it is a bound that k elements or more reach, and what reaches it (about k for values in no order) is ranked by
// counting.  Keys carry the value and, below it, the place: no two are equal, ties go to the lowest place by themselves.
// A second kernel, a block a group, adds up the sums of the parts, turns its beams' keys into totals and cuts them back in the same way.
// Parts' sums are added in 64 bits and totals compared in 64: with thousands of candidates, sums of 32 bits would order near ones
// by their rounding.
// Reordering: a thread owns 16 bytes of a row for all beams of a group and loads what they become before it stores the first.
#include "common.cuh"

namespace b200 {

constexpr int BEAM_THREADS = 512;
constexpr int BEAM_VEC = 8;                               // elements a thread takes of a tile
constexpr int BEAM_TILE = BEAM_THREADS * BEAM_VEC;
constexpr int BEAM_SLACK = 1024;                          // the list is cut back when it holds more than this
constexpr int BEAM_ROOM = BEAM_TILE + BEAM_SLACK;         // a tile more always fits
constexpr int BEAM_MOST = 256;                            // k at most
constexpr float kBeamLog2e = 1.4426950408889634f;

struct SelectArgs {
  const void* logits;
  const float* scores;           // [groups, width]
  uint64_t* keys;                // [rows, parts, k] best first
  int* counts;                   // [rows, parts]
  float* maxima;                 // [rows, parts]
  double* sums;                  // [rows, parts] of exp(x - maximum)
  float* out_scores;             // [groups, k]
  int* out_parents;
  long* out_tokens;
  int* status;
  cudaStream_t stream;
  long row_stride;
  int groups, width, vocab, k, parts, per_part, fp32;
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

template <typename Key>
struct BeamList {
  Key keys[BEAM_ROOM];
  Key slices[BEAM_THREADS];
  Key bound;
  int count;
};

// Cuts the list back to its k best, best first.  All threads of the block; the list has been written before a barrier.
template <typename Key>
__device__ void cut_back(BeamList<Key>& list, int k) {
  constexpr int PER = (BEAM_ROOM + BEAM_THREADS - 1) / BEAM_THREADS;
  const int tid = threadIdx.x;
  int n = list.count;
  int lanes = 32;                                         // lanes of a slice
  while (BEAM_THREADS / lanes < 2 * k && lanes > 1) lanes >>= 1;
  const int slices = BEAM_THREADS / lanes;
  // Only k slices reach the bound, and 2 k slices share the threads: a pass leaves 256 elements at most for every element that a thread
  // holds, 2560, 1280, 768, 512, 256 in turn; values in no order take one pass.
  while (n > max(3 * k, 256)) {
    Key mine[PER], top = Key::none();
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int at = tid + i * BEAM_THREADS;
      mine[i] = at < n ? list.keys[at] : Key::none();
      if (mine[i].above(top)) top = mine[i];
    }
    for (int o = 1; o < lanes; o <<= 1) {
      const Key other = top.other_lane(o);
      if (other.above(top)) top = other;
    }
    if (tid % lanes == 0) list.slices[tid / lanes] = top;
    if (tid == 0) list.bound = Key::none();
    __syncthreads();
    if (tid < slices) {
      const Key own = list.slices[tid];
      int rank = 0;
      for (int j = 0; j < slices; j++) rank += list.slices[j].above(own);
      if (rank == k - 1) list.bound = own;                // one thread, but for slices without an element: all of them none
    }
    if (tid == 0) list.count = 0;
    __syncthreads();
    const Key bound = list.bound;
#pragma unroll
    for (int i = 0; i < PER; i++)
      if (mine[i].above(Key::none()) && !bound.above(mine[i])) list.keys[atomicAdd(&list.count, 1)] = mine[i];
    __syncthreads();
    n = list.count;
    __syncthreads();
  }
  // rank by counting: 3 k elements at most
  static_assert(3 * BEAM_MOST <= 2 * BEAM_THREADS, "two elements a thread");
  Key own[2];
  int rank[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int at = tid + i * BEAM_THREADS;
    rank[i] = k;
    if (at < n) {
      own[i] = list.keys[at];
      rank[i] = 0;
      for (int j = 0; j < n; j++) rank[i] += list.keys[j].above(own[i]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; i++)
    if (rank[i] < k) list.keys[rank[i]] = own[i];
  if (tid == 0) list.count = min(n, k);
  __syncthreads();
}

// ---------------------------------------------------------------- parts of rows
__device__ __forceinline__ float beam_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ void load8(const T* at, float* x) {
  if constexpr (sizeof(T) == 2) {
    const uint4 r = __ldg(reinterpret_cast<const uint4*>(at));
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    const float4 a = __ldg(reinterpret_cast<const float4*>(at)), b = __ldg(reinterpret_cast<const float4*>(at) + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
}

__device__ __forceinline__ bool is_score(float s) { return s > -INFINITY && s < INFINITY; }

template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS, 2) select_rows_kernel(const SelectArgs a) {
  extern __shared__ __align__(16) uint8_t beam_smem[];
  BeamList<RowKey>& list = *reinterpret_cast<BeamList<RowKey>*>(beam_smem);
  __shared__ float warp_max[BEAM_THREADS / 32];
  __shared__ double warp_sum[BEAM_THREADS / 32];
  const int row = blockIdx.x / a.parts, part = blockIdx.x % a.parts, tid = threadIdx.x;
  if (!is_score(a.scores[row])) return;                  // the beam has ended: the second kernel asks its score first
  const T* x0 = (const T*)a.logits + (long)row * a.row_stride;
  // vectors lie on 16-byte boundaries of memory, whatever the row's first element does; a vector holds elements [at, at + 8)
  const int shift = (int)(((uintptr_t)x0 & 15) / sizeof(T));
  const int from = part * a.per_part - shift, to = min(from + a.per_part, a.vocab);
  float m = -INFINITY, s = 0.f, least = -INFINITY;
  if (tid == 0) list.count = 0;
  __syncthreads();
  auto fetch = [&](int at, float* x) {
    if (at >= 0 && at + BEAM_VEC <= a.vocab) {
      load8(x0 + at, x);
    } else {
#pragma unroll
      for (int j = 0; j < BEAM_VEC; j++) x[j] = at + j >= 0 && at + j < a.vocab ? (float)x0[at + j] : -INFINITY;
    }
  };
  float next[BEAM_VEC];
  int at = from + tid * BEAM_VEC;
  if (at < to) fetch(at, next);
  bool first = true;
  for (int base = from; base < to; base += BEAM_TILE, at += BEAM_TILE) {
    float x[BEAM_VEC];
#pragma unroll
    for (int j = 0; j < BEAM_VEC; j++) x[j] = next[j];
    const bool mine = at < to;
    if (at + BEAM_TILE < to) fetch(at + BEAM_TILE, next);
    bool over = false;
    if (mine) {
      float top = x[0];
#pragma unroll
      for (int j = 1; j < BEAM_VEC; j++) top = fmaxf(top, x[j]);
      if (top > m) {
        s *= beam_exp2((m - top) * kBeamLog2e);          // nothing before the first element that is above -inf
        m = top;
      }
      // differences from the maximum are taken before the factor: a product of the maximum would carry its rounding into every term
      const float under = m == -INFINITY ? 0.f : m;
      float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < BEAM_VEC; j++) t[j & 3] += beam_exp2((x[j] - under) * kBeamLog2e);       // a NaN or +inf: NaN
      s += (t[0] + t[1]) + (t[2] + t[3]);
      if (first) {
#pragma unroll
        for (int j = 0; j < BEAM_VEC; j++)
          if (at + j >= 0 && at + j < a.vocab)
            list.keys[atomicAdd(&list.count, 1)].v = ((uint64_t)order32(x[j]) << 32) | (uint32_t)~(at + j);
      } else if (top > least) {
#pragma unroll
        for (int j = 0; j < BEAM_VEC; j++)
          if (x[j] > least && at + j < a.vocab) {
            const int place = atomicAdd(&list.count, 1);
            list.keys[place].v = ((uint64_t)order32(x[j]) << 32) | (uint32_t)~(at + j);
            over |= place >= BEAM_SLACK;
          }
      }
    }
    if (__syncthreads_or(over) || first) {
      cut_back(list, a.k);
      if (list.count == a.k) least = unorder32((uint32_t)(list.keys[a.k - 1].v >> 32));
      __syncthreads();
    }
    first = false;
  }
  if (list.count > a.k) cut_back(list, a.k);
  const long slot = (long)row * a.parts + part;
  for (int i = tid; i < list.count; i += BEAM_THREADS) a.keys[slot * a.k + i] = list.keys[i].v;
  // the part's maximum and its sum under it
  float top = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((tid & 31) == 0) warp_max[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < BEAM_THREADS / 32; i++) top = fmaxf(top, warp_max[i]);
  double sum = m == -INFINITY ? (double)s : (double)s * (double)beam_exp2((m - top) * kBeamLog2e);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((tid & 31) == 0) warp_sum[tid >> 5] = sum;
  __syncthreads();
  if (tid == 0) {
    sum = 0.0;
    for (int i = 0; i < BEAM_THREADS / 32; i++) sum += warp_sum[i];
    a.maxima[slot] = top;
    a.sums[slot] = sum;
    a.counts[slot] = list.count;
  }
}

// ---------------------------------------------------------------- groups
__global__ void __launch_bounds__(BEAM_THREADS, 1) select_groups_kernel(const SelectArgs a) {
  extern __shared__ __align__(16) uint8_t beam_smem[];
  BeamList<GroupKey>& list = *reinterpret_cast<BeamList<GroupKey>*>(beam_smem);
  double* norm = reinterpret_cast<double*>(beam_smem + sizeof(BeamList<GroupKey>));      // log of a beam's sum; NaN: it has no candidates
  const int g = blockIdx.x, tid = threadIdx.x;
  for (int w = tid; w < a.width; w += BEAM_THREADS) {
    const long row = (long)g * a.width + w;
    double l = __longlong_as_double(0x7ff8000000000000ll);
    if (is_score(a.scores[row])) {
      float top = -INFINITY;
      for (int p = 0; p < a.parts; p++) top = fmaxf(top, a.maxima[row * a.parts + p]);
      double sum = 0.0;
      for (int p = 0; p < a.parts; p++) {
        const float mp = a.maxima[row * a.parts + p];
        const double sp = a.sums[row * a.parts + p];
        sum += mp == -INFINITY ? sp : sp * exp((double)mp - (double)top);
      }
      if (top > -INFINITY && top < INFINITY && sum > 0.0 && sum < 1e300) l = (double)top + log(sum);      // NaN fails both
    }
    norm[w] = l;
  }
  if (tid == 0) list.count = 0;
  __syncthreads();
  // candidates [beam, part, place in its list]; a beam without a distribution offers its first tokens at -inf
  const int per_beam = a.parts * a.k, all = a.width * per_beam;
  GroupKey least = GroupKey::none();
  for (int base = 0; base < all; base += BEAM_TILE) {
    for (int i = base + tid; i < min(base + BEAM_TILE, all); i += BEAM_THREADS) {
      const int w = i / per_beam, j = i - w * per_beam, p = j / a.k, c = j - p * a.k;
      const long row = (long)g * a.width + w, slot = row * a.parts + p;
      const double l = norm[w];
      GroupKey key = GroupKey::none();
      if (l != l) {
        if (p == 0 && c < a.vocab) key = {order64(-INFINITY), ~(uint32_t)(w * a.vocab + c)};
      } else if (c < a.counts[slot]) {
        const uint64_t r = a.keys[slot * a.k + c];
        const float x = unorder32((uint32_t)(r >> 32));
        key = {order64((double)a.scores[row] + ((double)x - l)), ~((uint32_t)(w * a.vocab) + ~(uint32_t)r)};
      }
      if (key.above(least)) list.keys[atomicAdd(&list.count, 1)] = key;
    }
    __syncthreads();
    if (list.count > BEAM_SLACK || base + BEAM_TILE >= all) {
      cut_back(list, a.k);
      if (list.count == a.k) least = list.keys[a.k - 1];
    }
    __syncthreads();
  }
  for (int i = tid; i < a.k; i += BEAM_THREADS) {
    const GroupKey key = list.keys[i];
    const uint32_t place = ~key.place;
    const long to = (long)g * a.k + i;
    a.out_scores[to] = (float)unorder64(key.v);
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
  int num_tensors, groups, beams, chunks;
};

template <int BYTES>
struct Bits;
template <> struct Bits<16> { using type = uint4; };
template <> struct Bits<8> { using type = uint2; };
template <> struct Bits<4> { using type = uint32_t; };
template <> struct Bits<2> { using type = uint16_t; };
template <> struct Bits<1> { using type = uint8_t; };

constexpr int REORDER_BEAMS = 1024;        // beams of a group at most

// Elements [first, first + blockDim) of every row that moves: all loads, then all stores.  Up to MOST beams stay in registers; with
// MOST = 0 a thread's loads go to its column of shared memory (cp.async where 16 bytes move at once).
template <int BYTES, int MOST>
__device__ __forceinline__ void move_rows(const BeamTensor& t, const int* from, const int* to, int beams, long offset, uint8_t* stage) {
  using V = typename Bits<BYTES>::type;
  uint8_t* at = t.base + offset;
  if constexpr (MOST > 0) {
    V v[MOST];
#pragma unroll
    for (int w = 0; w < MOST; w++)
      if (w < beams && from[w] >= 0) v[w] = *reinterpret_cast<const V*>(at + (long)from[w] * t.row_stride);
#pragma unroll
    for (int w = 0; w < MOST; w++)
      if (w < beams && from[w] >= 0) *reinterpret_cast<V*>(at + (long)to[w] * t.row_stride) = v[w];
  } else {
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
}

template <int MOST>
__global__ void __launch_bounds__(256, MOST == 16 ? 1 : (MOST == 8 ? 2 : 4)) reorder_kernel(const ReorderArgs a) {
  extern __shared__ __align__(16) uint8_t beam_smem[];
  int* from = reinterpret_cast<int*>(beam_smem);         // row that a beam's row becomes; -1: it stays as it is
  int* to = from + a.beams;
  uint8_t* stage = beam_smem + ((2 * a.beams * sizeof(int) + 15) & ~(size_t)15);
  const int g = blockIdx.z;
  const BeamTensor t = a.tensors[blockIdx.y];
  int units = t.units;
  if (t.unit_tokens > 0 && a.lengths) {
    const int len = max(0, a.lengths[g]);
    units = min(units, (len + t.unit_tokens - 1) / t.unit_tokens);
  }
  const long run = (long)units * t.unit_bytes / t.width, all = run * t.outer;       // elements of a run, of a row
  if ((long)blockIdx.x * blockDim.x >= all) return;
  bool any = false;
  for (int w = threadIdx.x; w < a.beams; w += blockDim.x) {
    const long b = (long)g * a.beams;
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
  if (!__syncthreads_or(any)) return;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (long)gridDim.x * blockDim.x) {
    const long o = i / run, offset = o * t.outer_stride + (i - o * run) * t.width;
    switch (t.width) {
      case 16: move_rows<16, MOST>(t, from, to, a.beams, offset, stage); break;
      case 8: move_rows<8, MOST>(t, from, to, a.beams, offset, stage); break;
      case 4: move_rows<4, MOST>(t, from, to, a.beams, offset, stage); break;
      case 2: move_rows<2, MOST>(t, from, to, a.beams, offset, stage); break;
      default: move_rows<1, MOST>(t, from, to, a.beams, offset, stage); break;
    }
  }
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
  if (a.parts < 1 || a.per_part < BEAM_VEC || a.per_part % BEAM_VEC || (long)a.parts * a.per_part > 0x7fffffffL - BEAM_TILE ||
      (long)a.parts * a.per_part < (long)a.vocab + BEAM_VEC - 1)
    return 9932;
  const int row_smem = (int)sizeof(BeamList<RowKey>), group_smem = (int)sizeof(BeamList<GroupKey>) + a.width * 8;
  if (group_smem > 200 * 1024) return 9933;
  const unsigned grid = (unsigned)(rows * a.parts);
  cudaError_t e = a.fp32 ? allow_smem<&select_rows_kernel<float>>(row_smem) : allow_smem<&select_rows_kernel<__nv_bfloat16>>(row_smem);
  if (e == cudaSuccess) e = allow_smem<&select_groups_kernel>(200 * 1024);
  if (e != cudaSuccess) return (int)e;
  if (a.fp32) select_rows_kernel<float><<<grid, BEAM_THREADS, row_smem, a.stream>>>(a);
  else select_rows_kernel<__nv_bfloat16><<<grid, BEAM_THREADS, row_smem, a.stream>>>(a);
  int rc = B200_CHECK_LAUNCH();
  if (rc) return rc;
  select_groups_kernel<<<a.groups, BEAM_THREADS, group_smem, a.stream>>>(a);
  return B200_CHECK_LAUNCH();
}

B200_API int b200_beam_reorder(const b200::ReorderArgs* args) {
  using namespace b200;
  const ReorderArgs& a = *args;
  if (a.groups <= 0 || a.beams <= 0 || a.num_tensors <= 0 || a.chunks <= 0) return 0;
  if (a.beams > REORDER_BEAMS || a.groups > 65535 || a.num_tensors > 65535) return 9940;
  const dim3 grid((unsigned)a.chunks, (unsigned)a.num_tensors, (unsigned)a.groups);
  const int lists = (2 * a.beams * 4 + 15) & ~15;
  if (a.beams <= 4) reorder_kernel<4><<<grid, 256, lists, a.stream>>>(a);
  else if (a.beams <= 8) reorder_kernel<8><<<grid, 256, lists, a.stream>>>(a);
  else if (a.beams <= 16) reorder_kernel<16><<<grid, 256, lists, a.stream>>>(a);
  else {
    // 32 threads of up to 128 beams, fewer of more: a block's columns stay within 64 KB
    const int threads = a.beams <= 128 ? 32 : (a.beams <= 256 ? 16 : (a.beams <= 512 ? 8 : 4));
    const int smem = lists + a.beams * threads * 16;
    const cudaError_t e = allow_smem<&reorder_kernel<0>>(80 * 1024);
    if (e != cudaSuccess) return (int)e;
    reorder_kernel<0><<<grid, threads, smem, a.stream>>>(a);
  }
  return B200_CHECK_LAUNCH();
}
