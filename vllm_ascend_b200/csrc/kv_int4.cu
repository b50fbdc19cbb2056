// Rows of keys and values into a 4-bit cache and back (format: kv_int4.cuh).
//
// Bound: memory.  A thread takes 8 channels of a row (16 bytes dense, 4 packed), four threads share a group and find its
// largest magnitude as whole numbers (the bits of |bf16| order as its values do, NaN and infinities above all numbers).
#include "kv_int4.cuh"

namespace b200 {

struct Kv4Rows {
  void *k, *v;                    // [rows, heads, D] bf16, heads dense; written by the read
  uint8_t *k_cache, *v_cache;
  const long long* slots;
  long k_stride, v_stride, rows, num_slots;
  int heads, D, block_size;
  int* status;
};

// x / s for a group's scale, to the nearest whole number, ties to even.  With 8 significant bits of x and 5 of s a quotient that is no
// tie lies at least 2^-11 from one, so the product with the reciprocal (off by less than 2^-20) is first rounded to a multiple of
// 2^-13, which puts ties back where they are.
__device__ __forceinline__ uint32_t kv4_code(float x, float r) {
  const float q = fmaf(x, r, 1536.f) - 1536.f;
  return __float_as_uint(q + 12582920.f) & 15u;      // 1.5 2^23 + 8
}

template <bool WRITE>
__global__ void __launch_bounds__(256) kv4_rows_kernel(const Kv4Rows p) {
  const int per_head = p.D >> 3, per_row = p.heads * per_head;
  const long first = (long)blockIdx.x * 256;
  const long row0 = first / per_row;                           // the same in all threads
  const int in_row = (int)(first - row0 * per_row) + threadIdx.x;
  const long row = row0 + in_row / per_row;
  const int item = in_row % per_row, h = item / per_head, c8 = item - h * per_head;
  const bool here = row < p.rows;
  const bool keys = blockIdx.y == 0;
  const long long slot = here ? p.slots[row] : -1;
  const bool stored = slot >= 0 && slot < p.num_slots;
  if (here && slot >= p.num_slots && p.status) atomicExch(p.status, B200_BAD_INDEX);
  uint8_t* unit = nullptr;
  int t = 0;
  if (stored) {
    const long blk = slot / p.block_size;
    const int off = (int)(slot - blk * p.block_size);
    t = off % KV4_TOKENS;
    unit = (keys ? p.k_cache : p.v_cache) +
           ((blk * p.heads + h) * (p.block_size / KV4_TOKENS) + off / KV4_TOKENS) * (long)kv4_unit_bytes(p.D);
  }
  const int data = keys ? kv4_key_word(p.D, t, c8 * 8) : kv4_value_word(p.D, t, c8 * 8) + 2 * (t & 1);
  const int scale = kv4_scale(p.D, t, c8 >> 2);
  __nv_bfloat16* dense = (__nv_bfloat16*)(keys ? p.k : p.v) + row * (keys ? p.k_stride : p.v_stride) + h * p.D + c8 * 8;
  if (WRITE) {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (stored) x = *reinterpret_cast<const uint4*>(dense);
    uint32_t top = __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
    top = max(top & 0xffffu, top >> 16);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));      // groups of four lanes: a row has a multiple of four items
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    if (!stored) return;
    uint32_t word = 0x88888888u, s16 = 0;
    if (top >= 0x7f80u) {
      s16 = 0x7fc0u;                                           // not finite: the whole group is NaN
    } else if (top > 0) {
      uint32_t sb = (__float_as_uint(__fdiv_rn(__uint_as_float(top << 16), 7.f)) + 0x7ffffu) & ~0x7ffffu;
      sb = min(max(sb, 0x17800000u), 0x51800000u);             // 2^-80 and 2^36; larger magnitudes saturate
      s16 = sb >> 16;
      const float s = __uint_as_float(sb);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
      word = 0;
      if (sb < 0x51800000u) {
        const float r = 1.f / s;
#pragma unroll
        for (int i = 0; i < 4; i++)
          word |= kv4_code(__uint_as_float(w[i] << 16), r) << (8 * i) | kv4_code(__uint_as_float(w[i] & 0xffff0000u), r) << (8 * i + 4);
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float v = __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
          const int n = (int)rintf(fminf(fmaxf(__fdiv_rn(v, s), -7.f), 7.f));
          word |= (uint32_t)(n + 8) << (4 * i);
        }
      }
    }
    if (keys) {
      *reinterpret_cast<uint32_t*>(unit + data) = word;
    } else {
      *reinterpret_cast<uint16_t*>(unit + data) = (uint16_t)word;
      *reinterpret_cast<uint16_t*>(unit + data + 4) = (uint16_t)(word >> 16);
    }
    if ((c8 & 3) == 0) *reinterpret_cast<uint16_t*>(unit + scale) = (uint16_t)s16;
  } else {
    if (!here) return;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (stored) {
      const uint32_t w = keys ? *reinterpret_cast<const uint32_t*>(unit + data)
                              : *reinterpret_cast<const uint16_t*>(unit + data) | (uint32_t)*reinterpret_cast<const uint16_t*>(unit + data + 4) << 16;
      const float s = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(unit + scale) << 16);
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; i++)
        o[i] = pack_bf16x2((float)((int)(w >> (8 * i) & 15u) - 8) * s, (float)((int)(w >> (8 * i + 4) & 15u) - 8) * s);
      x = make_uint4(o[0], o[1], o[2], o[3]);
    }
    *reinterpret_cast<uint4*>(dense) = x;
  }
}

static int kv4_rows(bool write, const Kv4Rows& p, cudaStream_t stream) {
  if (p.rows <= 0) return 0;
  if ((p.D != 64 && p.D != 128) || p.heads < 1 || p.heads > 4096 || p.block_size < KV4_TOKENS || p.block_size % KV4_TOKENS) return 9880;
  if ((p.k_stride & 7) || (p.v_stride & 7)) return 9881;
  const long blocks = (p.rows * p.heads * (p.D >> 3) + 255) / 256;
  if (blocks > 0x7fffffffl) return 9882;
  const dim3 grid((unsigned)blocks, 2);
  if (write) kv4_rows_kernel<true><<<grid, 256, 0, stream>>>(p);
  else kv4_rows_kernel<false><<<grid, 256, 0, stream>>>(p);
  return B200_CHECK_LAUNCH();
}

}  // namespace b200

using namespace b200;

// rows of k and v [rows, heads, D] (bf16, row strides given) into the slots of a 4-bit cache; slots below zero are skipped
B200_API int b200_kv_int4_write(const void* k, long k_stride, const void* v, long v_stride, long rows, const void* slots, void* k_cache,
                                void* v_cache, long num_slots, int heads, int D, int block_size, int* status, cudaStream_t stream) {
  Kv4Rows p = {const_cast<void*>(k), const_cast<void*>(v), (uint8_t*)k_cache, (uint8_t*)v_cache, (const long long*)slots, k_stride, v_stride,
               rows, num_slots, heads, D, block_size, status};
  return kv4_rows(true, p, stream);
}

// the rows of slots as dense bf16 [rows, heads, D]; slots below zero read as zeros
B200_API int b200_kv_int4_read(void* k, void* v, long rows, const void* slots, const void* k_cache, const void* v_cache, long num_slots,
                               int heads, int D, int block_size, int* status, cudaStream_t stream) {
  const long stride = (long)heads * D;
  Kv4Rows p = {k, v, (uint8_t*)const_cast<void*>(k_cache), (uint8_t*)const_cast<void*>(v_cache), (const long long*)slots, stride, stride,
               rows, num_slots, heads, D, block_size, status};
  return kv4_rows(false, p, stream);
}
