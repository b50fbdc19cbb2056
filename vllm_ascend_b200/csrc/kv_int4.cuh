// Keys and values in 4 bits: how a page lies in memory, and how it is unpacked.
//
// Groups of 32 adjacent channels of a (token, head) share a scale s: the smallest number of five significant bits with
// 7 s no less than the group's largest magnitude, between 2^-80 and 2^34, held as bf16.  A channel x is the whole number
// n = rint(x / s) (ties to even), -7..7, held as n + 8, and stands for n s, three bits times five: exact in bf16.
//
// A bf16 whose low byte alone is set has the value (low byte) 2^-133, through subnormals and the first exponent alike.  So a nibble that
// a mask leaves in either half of a low byte is a number as it stands, and one packed multiply-add makes two channels of it:
// (n + 8) 2^-133 * 2^93 s - 2^-37 s = n s 2^-40 (the upper half of a byte: 2^89 s).  A word of eight channels takes five integer
// instructions, where shifting each nibble below the leading one of 16 takes eight.  The factor 2^-40 keeps 2^93 s within bf16; the
// kernels undo it in fp32.
//
// A cache is [blocks][heads][block size / 16 units], a unit 9 D bytes for 16 tokens, in one run, so that a tile of a head is
// fetched by one bulk copy.  A word holds eight adjacent channels, the lower of two in the lower nibble.
//   keys    16 rows of D / 2 bytes, a token each, words in order
//   values  8 rows of D bytes, a pair of tokens each: chunks of 16 bytes for 16 channels, each word two bytes of the even token and
//           two of the odd one (what a lane of the second product needs, side by side), chunk x at x ^ kv4_value_swizzle(row) so
//           that lanes with different rows meet in different banks
// and behind either D / 32 x 16 scales (bf16), group by group, tokens in order.
#pragma once
#include "common.cuh"

namespace b200 {

constexpr int KV4_TOKENS = 16;      // of a unit
constexpr int KV4_GROUP = 32;       // channels of a scale
__host__ __device__ constexpr int kv4_unit_bytes(int D) { return 9 * D; }
__host__ __device__ constexpr int kv4_value_swizzle(int D, int pair) { return D == 128 ? 2 * (pair & 3) : pair & 2; }
// bytes within a unit: the word of a token's keys that holds channels ch .. ch + 7; that whose half holds ch .. ch + 3 of its values
__host__ __device__ constexpr int kv4_key_word(int D, int t, int ch) { return t * (D / 2) + ch / 2; }
__host__ __device__ constexpr int kv4_value_word(int D, int t, int ch) {
  return (t >> 1) * D + (((ch >> 4) ^ kv4_value_swizzle(D, t >> 1)) << 4) + (ch & 12);
}
__host__ __device__ constexpr int kv4_scale(int D, int t, int g) { return 8 * D + 2 * (g * KV4_TOKENS + t); }

constexpr float KV4_UNDO = 1099511627776.f;      // 2^40

// A scale (a pair of them, of what lies in the halves of a word) as multipliers and summand.
struct Kv4Scale {
  __nv_bfloat162 low, high, minus;
  __device__ __forceinline__ explicit Kv4Scale(uint32_t pair) {
    const __nv_bfloat162 s = *reinterpret_cast<const __nv_bfloat162*>(&pair);
    low = __hmul2(s, __floats2bfloat162_rn(0x1p93f, 0x1p93f));
    high = __hmul2(s, __floats2bfloat162_rn(0x1p89f, 0x1p89f));
    minus = __hmul2(s, __floats2bfloat162_rn(-0x1p-37f, -0x1p-37f));
  }
};
// nibble 0 or 1 of the halves' low bytes: n s 2^-40
__device__ __forceinline__ uint32_t kv4_pair(int nibble, uint32_t w, const Kv4Scale& s) {
  uint32_t m = w & (nibble ? 0x00f000f0u : 0x000f000fu);
  const __nv_bfloat162 v = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&m), nibble ? s.high : s.low, s.minus);
  return *reinterpret_cast<const uint32_t*>(&v);
}

}  // namespace b200
