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
  long q_stride, out_stride, num_blocks, q_rows;
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

// Checks and fills what both kernels take; 0 or an error code.
int int4_params(Int4Params* p, const void* q, long q_stride, long q_rows, const void* k_cache, const void* v_cache, long num_blocks, int block_size,
                const void* cu, const void* seq_lens, const void* block_table, int max_blocks, int num_seqs, int Hq, int Hkv, int D,
                float scale, int causal, int window, int parts, void* out, long out_stride, void* scratch, int* status);
int int4_join(const Int4Params& p, int D, long q_rows, cudaStream_t stream);

}  // namespace b200
