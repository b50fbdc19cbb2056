// Keys and values in 4 bits: how a page lies in memory.
//
// Groups of 32 adjacent channels of a (token, head) share a scale s: the smallest number of five significant bits with
// 7 s no less than the group's largest magnitude, held as bf16.  A channel x is the whole number n = rint(x / s) (ties to even), -7..7,
// held as n + 8, and stands for n s, three bits times five: exact in bf16.  So is 24 s, which lets one packed
// multiply-add unpack two channels: a nibble put below the leading one of 16 reads 16 + (n + 8), and (24 + n) s - 24 s = n s.
//
// A cache is [blocks][heads][block size / 16 units], a unit 9 D bytes for 16 tokens, in one run, so that a tile of a head is
// fetched by one bulk copy a unit:
//   16 rows of D / 2 bytes   channel c of a row in nibble c % 2 (low first) of byte c / 2.  Keys: row = token % 16.  Values: even tokens
//                            of each eight first (kv4_value_row): a tensor-core lane takes tokens 2 i and 2 i + 1, and four lanes' rows
//                            are then adjacent
//   D / 32 x 16 bf16         scales, group by group, tokens in order: what pairs of tokens need is one word
#pragma once
#include "common.cuh"

namespace b200 {

constexpr int KV4_TOKENS = 16;      // of a unit
constexpr int KV4_GROUP = 32;       // channels of a scale
__host__ __device__ constexpr int kv4_unit_bytes(int D) { return 9 * D; }
__host__ __device__ constexpr int kv4_value_row(int t) { return (t & 8) | ((t & 1) << 2) | ((t >> 1) & 3); }

// two nibbles of a word (bits 4 j of either half) next to a scale: bf16 pairs n s.  s24 is -24 s.
template <int j>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t w, __nv_bfloat162 s, __nv_bfloat162 s24) {
  const uint32_t x = j == 0 ? w << 3 : w >> (4 * j - 3);
  uint32_t m = (x & 0x00780078u) | 0x41804180u;
  const __nv_bfloat162 v = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&m), s, s24);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ __nv_bfloat162 kv4_scale(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
__device__ __forceinline__ __nv_bfloat162 kv4_minus24(__nv_bfloat162 s) {
  return __hmul2(s, __floats2bfloat162_rn(-24.f, -24.f));
}

}  // namespace b200
