// A key/value cache held in 4 bits: the format, shared by the kernels that write it, read it back and attend to it.
//
// 32 dims of a head of one position are a group: a scale s and a zero z.  With lo = min(0, smallest), hi = max(0, largest),
//   s = (hi - lo) / 15 rounded up to a half-precision number of six significant bits, at most KV4_LARGEST,
//   z = rint(-lo / s),  n = rint(x / s) + z,  both kept in 0 .. 15,  and the number held is s (n - z):
// at most ten significant bits (six by four), so half precision has every number of the cache exactly, and so do the matrix
// cores.  |x - s (n - z)| <= s / 2 where the range fits (hi - lo <= 31,680); beyond it numbers saturate.  A group that holds a
// number that is not finite reads NaN throughout.  A scale's word of 16 bits is the half-precision number's (its low five bits
// are zero) with z in the low four.
//
// A word of 32 bits holds eight numbers e0 .. e7: the sum of e(2i) << 4i and e(2i+1) << (16 + 4i), rotated left by 6.  Rotated
// right by 4i, bits 6..9 and 22..25 are e(2i) and e(2i+1): with 0x4C00 in either half the half-precision pair 16 + e, without a
// shift for the first pair, and one packed multiply-add makes the two numbers of it: (16 + e) s - (16 + z) s, exactly.
//
// Keys:   [page][kv head]: [slot][HD / 8] words (of eight dims), then [slot][HD / 32] scales.
// Values: [page][kv head]: [slot / 8][HD] words (of one dim's eight positions), then [slot / 8][HD / 32][8] scales: the
// operands of the value product want consecutive positions of a dim.
#pragma once

#include "common.h"

#define KV4_LARGEST 2112.0f        // 31 s has to be finite in half precision: (16 + z) s is taken off
#define KV4_NAN 0x7FE0             // the scale of a group that is not finite

typedef __attribute__((ext_vector_type(2))) _Float16 half2_t;

__host__ __device__ inline int kv4_row_bytes(int head_dim) { return head_dim / 2 + head_dim / 16; }

// Sizes that the 4-bit cache's kernels take: pages whose place is a shift, octets of values inside a page.
__host__ inline bool kv4_takes(int head_dim, int page_size) {
  return (head_dim == 64 || head_dim == 128) && page_size >= 8 && page_size <= 1024 && (page_size & (page_size - 1)) == 0;
}

__host__ __device__ inline int kv4_place(int i) { return (6 + 4 * (i >> 1) + 16 * (i & 1)) & 31; }   // the lowest bit of number i

// A scale's half-precision bits for a group's range hi - lo.
__device__ inline int kv4_scale_bits(float range) {
  const float want = fminf(__fdiv_rn(range, 15.0f), KV4_LARGEST);
  float s;
  if (want < 0x1p-14f) {
    s = __fmul_rn(ceilf(__fmul_rn(want, 0x1p19f)), 0x1p-19f);            // half precision's steps below its smallest normal
  } else {
    s = __uint_as_float((__float_as_uint(want) + 0x3FFFFu) & ~0x3FFFFu);   // five bits behind the leading one, upwards
  }
  const _Float16 h = (_Float16)s;                                          // exact
  return __builtin_bit_cast(unsigned short, h);
}

__device__ inline float kv4_scale_of(unsigned meta) {
  return (float)__builtin_bit_cast(_Float16, (unsigned short)(meta & 0x7FE0));
}

// The constants of the unpacking, in registers: as constants the compiler takes two instructions for both masks, not one.
struct Kv4Masks {
  unsigned digit, sixteens;
};
__device__ __forceinline__ Kv4Masks kv4_masks() {
  Kv4Masks m = {0x03C003C0u, 0x4C004C00u};
  asm("" : "+s"(m.digit));
  asm("" : "+v"(m.sixteens));
  return m;
}

// A word's eight numbers as an operand of the matrix cores; s and c hold the scales and -(16 + z) s of each pair.  Eleven
// instructions for eight numbers: three rotations, four times both masks, four packed multiply-adds.
__device__ __forceinline__ u32x4 kv4_operand(unsigned word, const half2_t (&s)[4], const half2_t (&c)[4], const Kv4Masks& masks) {
  u32x4 out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned x = (__builtin_rotateright32(word, 4 * i) & masks.digit) | masks.sixteens;
    out[i] = __builtin_bit_cast(unsigned, __builtin_elementwise_fma(__builtin_bit_cast(half2_t, x), s[i], c[i]));
  }
  return out;
}

// The scales of two numbers, from a pair of scale words.
__device__ __forceinline__ void kv4_pair_scale(unsigned metas, half2_t& s, half2_t& c) {
  s = __builtin_bit_cast(half2_t, metas & 0x7FE07FE0u);
  c = -__builtin_bit_cast(half2_t, ((metas << 6) & 0x03C003C0u) | 0x4C004C00u) * s;
}

// One of an operand's two numbers, in 32 bits.
__device__ __forceinline__ float kv4_half(unsigned pair, int which) { return (float)__builtin_bit_cast(half2_t, pair)[which]; }
