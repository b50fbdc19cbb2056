// What the kernels of attention over a 4-bit cache share: arguments, parts of rows and how they join.
#pragma once
#include "kv_int4.cuh"

namespace b200 {

constexpr int I4_CLUSTER = 16;     // blocks of a cluster at most
constexpr int I4_PARTS = 64;       // parts at most

struct Int4Params {
  const __nv_bfloat16* q;
  const uint8_t *k_cache, *v_cache;
  const int *cu, *seq_lens, *block_table;
  __nv_bfloat16* out;
  float *part_o, *part_lse;       // [tokens x heads][parts][D], [..][parts]: results of parts, normalised, with log2 of their sums
  long q_stride, out_stride, table_stride, num_blocks, q_rows;
  int num_seqs, max_blocks, block_size, G, Hkv, parts, cluster, row_blocks, causal, window;
  uint32_t g_inv, upp_inv;        // ceil(2^32 / .) of G and of the units of a page (int4_div)
  float scale_log2;               // of scores over unpacked keys, which carry 2^-40
  int* status;
};

// x / d for x d < 2^32 with inv = ceil(2^32 / d)
__device__ __forceinline__ int int4_div(int x, int d, uint32_t inv) { return d == 1 ? x : (int)__umulhi((uint32_t)x, inv); }

__device__ __forceinline__ float i4_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void i4_bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// What the entry points take, by address: one argument instead of 25 saves their caller 2.4 us.
struct Int4Args {
  const void *q, *k_cache, *v_cache;
  const int *cu, *seq_lens, *block_table;
  void *out, *scratch;
  int* status;
  cudaStream_t stream;
  long q_stride, q_rows, num_blocks, out_stride, tokens, table_stride;
  float scale;
  int block_size, max_blocks, num_seqs, max_q_len, Hq, Hkv, D, causal, window, parts;
};
static_assert(sizeof(Int4Args) == 176, "pointers, longs and ints without gaps, as they are packed");

// Checks and fills what both kernels take; 0 or an error code.
int int4_params(Int4Params* p, const Int4Args& a);
int int4_join(const Int4Params& p, int D, long q_rows, cudaStream_t stream);

}  // namespace b200
