// Rows of keys and values into a 4-bit cache and back (format: kv_int4.cuh).
//
// Bound: memory, and for rows in the instructions that round them next to it.  A thread keeps to 8 channels (16 bytes dense, 4 packed) and
// walks rows, keys and values of two neighbouring rows in flight at once; what a row's slot means is found once for the block.  Four threads
// share a group and find its largest magnitude as whole numbers (the bits of |bf16| order as its values do, NaN and infinities
// above all numbers).
// Measured, 8 heads of 128: 96000 rows out of the cache 107 us (4.7 TB/s; writing the same dense bytes alone takes 102 us; 123 us with the
// rows of a thread apart, so that neighbouring ones are written at different times); 96000 rows in 103 us, 4.9 TB/s (129 us
// with values stored by twos of bytes, codes masked and shifted into place one by one, and products for every address); 8192
// rows 13 and 10 us; one row 2.4 us, a launch.
#include "kv_int4.cuh"

namespace b200 {

constexpr int KV4_ROWS_THREADS = 256;
constexpr int KV4_ROWS_MAX = 256;           // of a block
constexpr int KV4_FLIGHT = 2;               // rows of a thread whose loads are under way together

struct Kv4Rows {
  void *k, *v;                    // [rows, heads, D] bf16, heads dense; written by the read
  uint8_t *k_cache, *v_cache;
  const long long* slots;
  long k_stride, v_stride, rows, num_slots;
  int heads, D, block_size, rows_per_block;
  int* status;
};

// Two channels (the halves of w) over s, r its reciprocal, to the nearest whole numbers, ties to even: n as the bits of a float, KV4_ZERO
// more.  With 8 significant bits of x and 5 of s a quotient that is no tie lies at least 2^-11 from one, so the product with an
// approximate reciprocal (off by less than 2^-18) is first rounded to a multiple of 2^-13, which puts ties back where they are.
constexpr uint32_t KV4_ZERO = 0x4b400000u;             // 1.5 2^23
__device__ __forceinline__ uint2 kv4_codes(uint32_t w, float r) {
  uint2 n;
  asm("{\n\t.reg .b64 x, r, a, b;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 r, {%4, %4};\n\tmov.b64 a, {%5, %5};\n\tmov.b64 b, {%6, %6};\n\t"
      "fma.rn.f32x2 x, x, r, a;\n\tadd.rn.f32x2 x, x, b;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=r"(n.x), "=r"(n.y)
      : "r"(w << 16), "r"(w & 0xffff0000u), "f"(r), "f"(1536.f), "f"(12581376.f));       // 1.5 2^10, and what it lacks of 1.5 2^23
  return n;
}

// Eight channels (x) of a group to a word; s16 receives the group's scale as bf16.  All lanes of a warp call it.
__device__ __forceinline__ uint32_t kv4_quantise(const uint4& x, uint32_t& s16) {
  uint32_t top = __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
  top = max(top & 0xffffu, top >> 16);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  s16 = top >= 0x7f80u ? 0x7fc0u : 0u;                         // not finite: the whole group is NaN
  if (top == 0 || top >= 0x7f80u) return 0x88888888u;
  // top = m 2^(e - 134), m of eight bits; the smallest five-bit number from m / 7 on is ceil(m / 7) up to 31, an even one above
  const uint32_t e = top >> 7, m = (top & 0x7fu) | 0x80u;
  uint32_t k = ((m + 6) * 9363u) >> 16;
  if (k > 31) k = (((m + 13) * 4682u) >> 16) * 2;
  float s = __uint_as_float((e > 7 ? e - 7 : 1) << 23) * (float)k;
  s = fminf(fmaxf(s, 0x1p-80f), 0x1p34f);                      // larger magnitudes saturate
  s16 = __float_as_uint(s) >> 16;
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t word = 0;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  if (s < 0x1p34f) {
    // nibbles n + 8 from a sum of 16^i (KV4_ZERO + n): the constant parts go at the end
#pragma unroll
    for (int i = 3; i >= 0; i--) {
      const uint2 n = kv4_codes(w[i], r);
      word = (word * 16 + n.y) * 16 + n.x;
    }
    word -= 0x11111111u * (KV4_ZERO - 8u);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float v = __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
      word |= (uint32_t)((int)rintf(fminf(fmaxf(v * 0x1p-34f, -7.f), 7.f)) + 8) << (4 * i);
    }
  }
  return word;
}

// A word next to its scale as eight bf16 channels.
__device__ __forceinline__ uint4 kv4_unpack(uint32_t w, uint32_t s16) {
  const Kv4Scale s(s16 * 0x10001u);
  uint32_t v[4] = {kv4_pair(0, w, s), kv4_pair(1, w, s), kv4_pair(0, w >> 8, s), kv4_pair(1, w >> 8, s)};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const __nv_bfloat162 u = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v[i]), __floats2bfloat162_rn(KV4_UNDO, KV4_UNDO));
    v[i] = *reinterpret_cast<const uint32_t*>(&u);
  }
  return make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410), __byte_perm(v[0], v[1], 0x7632),
                    __byte_perm(v[2], v[3], 0x7632));
}

template <bool WRITE, int D, int U>
__global__ void __launch_bounds__(KV4_ROWS_THREADS) kv4_rows_kernel(const Kv4Rows p) {
  __shared__ long unit_of[KV4_ROWS_MAX];        // where the row's unit begins within head 0 of its block, token of the unit in the low bits; -1: none
  const long row0 = (long)blockIdx.x * p.rows_per_block;
  const int rows = (int)min((long)p.rows_per_block, p.rows - row0), upp = p.block_size / KV4_TOKENS;
  for (int i = threadIdx.x; i < rows; i += KV4_ROWS_THREADS) {
    const long long slot = p.slots[row0 + i];
    long at = -1;
    if (slot >= 0 && slot < p.num_slots) {
      const long blk = slot / p.block_size;
      const int off = (int)(slot - blk * p.block_size);
      at = (blk * p.heads * upp + off / KV4_TOKENS) * kv4_unit_bytes(D) + off % KV4_TOKENS;
      static_assert(kv4_unit_bytes(D) % KV4_TOKENS == 0, "");
    } else if (slot >= 0 && p.status) {
      atomicExch(p.status, B200_BAD_INDEX);
    }
    unit_of[i] = at;
  }
  __syncthreads();
  const int per_row = p.heads * (D / 8), together = max(1, KV4_ROWS_THREADS / per_row);        // items of a row, rows at once
  for (int item0 = 0; item0 < per_row; item0 += KV4_ROWS_THREADS) {
    const int sub = per_row > KV4_ROWS_THREADS ? 0 : threadIdx.x / per_row;
    const int item = per_row > KV4_ROWS_THREADS ? item0 + threadIdx.x : threadIdx.x - sub * per_row;
    const bool mine = sub < together && item < per_row;
    const int h = item / (D / 8), c8 = item - h * (D / 8);
    const long head = (long)h * upp * kv4_unit_bytes(D);
    const __nv_bfloat16 *ks = (const __nv_bfloat16*)p.k + h * D + c8 * 8, *vs = (const __nv_bfloat16*)p.v + h * D + c8 * 8;
    for (int i0 = 0; i0 < rows; i0 += U * together) {
      uint4 x[U][2];
      long at[U];
      uint32_t w[U][2], s16[U][2];
      const int first = i0 + sub * U;
      bool pair = false;                        // two tokens whose values lie side by side
      if constexpr (WRITE && U == 2) pair = mine && first + 1 < rows && !(unit_of[first] & 1) && unit_of[first + 1] == unit_of[first] + 1;
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int i = i0 + sub * U + u;
        at[u] = mine && i < rows ? unit_of[i] : -1;
        x[u][0] = x[u][1] = make_uint4(0, 0, 0, 0);
        w[u][0] = w[u][1] = s16[u][0] = s16[u][1] = 0;
        if (at[u] < 0) continue;
        if (WRITE) {
          x[u][0] = *reinterpret_cast<const uint4*>(ks + (row0 + i) * p.k_stride);
          x[u][1] = *reinterpret_cast<const uint4*>(vs + (row0 + i) * p.v_stride);
        } else {
          const int t = (int)(at[u] & (KV4_TOKENS - 1));
          const long unit = at[u] - t + head;
          const uint8_t *ku = p.k_cache + unit, *vu = p.v_cache + unit;
          const int vw = kv4_value_word(D, t, c8 * 8) + 2 * (t & 1), sc = kv4_scale(D, t, c8 >> 2);
          w[u][0] = *reinterpret_cast<const uint32_t*>(ku + kv4_key_word(D, t, c8 * 8));
          w[u][1] = *reinterpret_cast<const uint16_t*>(vu + vw) | (uint32_t)*reinterpret_cast<const uint16_t*>(vu + vw + 4) << 16;
          s16[u][0] = *reinterpret_cast<const uint16_t*>(ku + sc);
          s16[u][1] = *reinterpret_cast<const uint16_t*>(vu + sc);
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int i = i0 + sub * U + u;
        if (WRITE) {
#pragma unroll
          for (int kv = 0; kv < 2; kv++) w[u][kv] = kv4_quantise(x[u][kv], s16[u][kv]);
          if (at[u] < 0) continue;
          if (pair) {
            if (u == 0) continue;
            const int t = (int)(at[0] & (KV4_TOKENS - 1));
            const long unit = at[0] - t + head;
            uint8_t *ku = p.k_cache + unit, *vu = p.v_cache + unit;
            *reinterpret_cast<uint32_t*>(ku + kv4_key_word(D, t, c8 * 8)) = w[0][0];
            *reinterpret_cast<uint32_t*>(ku + kv4_key_word(D, t + 1, c8 * 8)) = w[U - 1][0];
            *reinterpret_cast<uint2*>(vu + kv4_value_word(D, t, c8 * 8)) =
                make_uint2(__byte_perm(w[0][1], w[U - 1][1], 0x5410), __byte_perm(w[0][1], w[U - 1][1], 0x7632));
            if ((c8 & 3) == 0) {
              *reinterpret_cast<uint32_t*>(ku + kv4_scale(D, t, c8 >> 2)) = s16[0][0] | s16[U - 1][0] << 16;
              *reinterpret_cast<uint32_t*>(vu + kv4_scale(D, t, c8 >> 2)) = s16[0][1] | s16[U - 1][1] << 16;
            }
            continue;
          }
          const int t = (int)(at[u] & (KV4_TOKENS - 1));
          const long unit = at[u] - t + head;
          uint8_t *ku = p.k_cache + unit, *vu = p.v_cache + unit;
          const int vw = kv4_value_word(D, t, c8 * 8) + 2 * (t & 1), sc = kv4_scale(D, t, c8 >> 2);
          *reinterpret_cast<uint32_t*>(ku + kv4_key_word(D, t, c8 * 8)) = w[u][0];
          *reinterpret_cast<uint16_t*>(vu + vw) = (uint16_t)w[u][1];
          *reinterpret_cast<uint16_t*>(vu + vw + 4) = (uint16_t)(w[u][1] >> 16);
          if ((c8 & 3) == 0) {
            *reinterpret_cast<uint16_t*>(ku + sc) = (uint16_t)s16[u][0];
            *reinterpret_cast<uint16_t*>(vu + sc) = (uint16_t)s16[u][1];
          }
        } else if (mine && i < rows) {
          uint4 *ko = (uint4*)((__nv_bfloat16*)p.k + (row0 + i) * p.k_stride + h * D + c8 * 8);
          uint4 *vo = (uint4*)((__nv_bfloat16*)p.v + (row0 + i) * p.v_stride + h * D + c8 * 8);
          *ko = at[u] < 0 ? make_uint4(0, 0, 0, 0) : kv4_unpack(w[u][0], s16[u][0]);
          *vo = at[u] < 0 ? make_uint4(0, 0, 0, 0) : kv4_unpack(w[u][1], s16[u][1]);
        }
      }
    }
  }
}

static int kv4_rows(bool write, Kv4Rows p, cudaStream_t stream) {
  if (p.rows <= 0) return 0;
  if ((p.D != 64 && p.D != 128) || p.heads < 1 || p.heads > 65536 || p.block_size < KV4_TOKENS || p.block_size % KV4_TOKENS) return 9880;
  if ((p.k_stride & 7) || (p.v_stride & 7)) return 9881;
  // KV4_FLIGHT rows a thread at least, more where that leaves eight blocks an SM; single rows where few are asked for
  const int per_row = p.heads * (p.D / 8), together = per_row < KV4_ROWS_THREADS ? KV4_ROWS_THREADS / per_row : 1;
  const bool many = p.rows >= (long)KV4_FLIGHT * together * num_sms();
  const int step = (many ? KV4_FLIGHT : 1) * together, most = KV4_ROWS_MAX / step > 0 ? KV4_ROWS_MAX / step : 1;
  long passes = p.rows / ((long)step * 8 * num_sms());
  passes = passes < 1 ? 1 : passes > most ? most : passes;
  p.rows_per_block = (int)(passes * step < KV4_ROWS_MAX ? passes * step : KV4_ROWS_MAX);
  const long blocks = (p.rows + p.rows_per_block - 1) / p.rows_per_block;
  if (blocks > 0x7fffffffl) return 9882;
  const unsigned g = (unsigned)blocks;
  const dim3 block(KV4_ROWS_THREADS);
#define KV4_ROWS(W, D, U) kv4_rows_kernel<W, D, U><<<g, block, 0, stream>>>(p)
  if (p.D == 128) {
    if (write) many ? KV4_ROWS(true, 128, KV4_FLIGHT) : KV4_ROWS(true, 128, 1);
    else many ? KV4_ROWS(false, 128, KV4_FLIGHT) : KV4_ROWS(false, 128, 1);
  } else {
    if (write) many ? KV4_ROWS(true, 64, KV4_FLIGHT) : KV4_ROWS(true, 64, 1);
    else many ? KV4_ROWS(false, 64, KV4_FLIGHT) : KV4_ROWS(false, 64, 1);
  }
#undef KV4_ROWS
  return B200_CHECK_LAUNCH();
}

}  // namespace b200

using namespace b200;

// by address, like attention's
struct Kv4Args {
  void *k, *v;
  const long long* slots;
  void *k_cache, *v_cache;
  int* status;
  cudaStream_t stream;
  long k_stride, v_stride, rows, num_slots;
  int heads, D, block_size;
};
static_assert(sizeof(Kv4Args) == 104, "pointers, longs and ints without gaps, as they are packed");
static Kv4Rows kv4_args(const Kv4Args& a) {
  return Kv4Rows{a.k, a.v, (uint8_t*)a.k_cache, (uint8_t*)a.v_cache, a.slots, a.k_stride, a.v_stride, a.rows, a.num_slots,
                 a.heads, a.D, a.block_size, 0, a.status};
}

// rows of k and v [rows, heads, D] (bf16, row strides given) into the slots of a 4-bit cache; slots below zero are skipped
B200_API int b200_kv_int4_write(const Kv4Args* a) { return kv4_rows(true, kv4_args(*a), a->stream); }

// the rows of slots as dense bf16 [rows, heads, D]; slots below zero read as zeros
B200_API int b200_kv_int4_read(const Kv4Args* a) { return kv4_rows(false, kv4_args(*a), a->stream); }
