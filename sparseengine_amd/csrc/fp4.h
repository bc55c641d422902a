// Keys and values held in 4 bits.
//
// 32 neighbouring dims of a key or of a value are a *group*: 32 codes of 4 bits and one byte for the group's
// factor.  A code is a sign (bit 3) and one of the eight magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6; the factor byte e
// stands for 2^(e - 127), and 255 says that the group is not a number (one of its elements was not finite).  This
// is the format the chip itself converts (two codes and a factor to two bfloat16 in one instruction, full rate:
// 1.85 ns per wavefront and instruction on MI355X, as much as any other), and every value it holds is a bfloat16
// exactly, so attention on a 4-bit cache is attention on a bfloat16 cache with those values.
//
// The factor of a group is the smallest 2^k, -125 <= k <= 125, with max |x| <= 7 * 2^k: the largest element is
// then off by no more than half a step of the largest two magnitudes (4 to 6), as any other, where the bound 6
// would take the next power of two, and with it half the resolution of all 32, for elements between 6 and 7.  The
// range of k keeps 0.5 * 2^k a normal float and 6 * 2^k finite.  The codes are the nearest magnitudes, ties to
// the even code (whose last bit is 0), magnitudes beyond 6 are 6.
//
// A cache layer is [pages, 2 (keys, values), kv_heads, page_size, head_dim * 17 / 32] bytes; a kv head's part of
// a page holds the codes, then the factors.  With G = head_dim / 32 groups, two codes to a byte (the even dim in
// the low half):
//   keys    codes [G][page_size][16 bytes]                    factors [G][page_size]
//   values  codes [page_size / 8][16][G][8]                   factors [page_size / 8][G][8]
//           (byte j of 16 holds dims 32 group + 2 j and + 1; the last index is the key within its eight)
// A lane of a matrix operand then reads one contiguous piece, and neighbouring lanes neighbouring pieces.
// head_dim % 32 == 0, page_size % 32 == 0: a step of 32 keys lies in one page, and every part of a page
// begins on a multiple of 16 bytes.
#pragma once
#include "common.h"

#define FP4_GROUP 32
#define FP4_NAN 255        // factor byte of a group that is not a number
#define FP4_MIN_EXP -125
#define FP4_MAX_EXP 125

__host__ __device__ __forceinline__ int64_t fp4_head_bytes(int page_size, int head_dim) {
  return static_cast<int64_t>(page_size) * (head_dim / 32) * 17;
}
__host__ __device__ __forceinline__ int64_t fp4_factors_at(int page_size, int head_dim) {
  return static_cast<int64_t>(page_size) * (head_dim / 2);
}
// offsets inside a kv head's part of a page
__host__ __device__ __forceinline__ int64_t fp4_key_code_at(int page_size, int off, int group) {
  return (static_cast<int64_t>(group) * page_size + off) * 16;        // + j: dims 2 j, 2 j + 1 of the group
}
__host__ __device__ __forceinline__ int64_t fp4_key_factor_at(int page_size, int head_dim, int off, int group) {
  return fp4_factors_at(page_size, head_dim) + static_cast<int64_t>(group) * page_size + off;
}
__host__ __device__ __forceinline__ int64_t fp4_value_code_at(int head_dim, int off, int group, int j) {
  return ((static_cast<int64_t>(off >> 3) * 16 + j) * (head_dim / 32) + group) * 8 + (off & 7);
}
__host__ __device__ __forceinline__ int64_t fp4_value_factor_at(int page_size, int head_dim, int off, int group) {
  return fp4_factors_at(page_size, head_dim) + (static_cast<int64_t>(off >> 3) * (head_dim / 32) + group) * 8 + (off & 7);
}

// The factor byte of a group whose largest magnitude is `amax` (not finite: FP4_NAN).
__device__ __forceinline__ int fp4_factor_of(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  if (bits >= 0x7f800000u) return FP4_NAN;
  // amax = m * 2^k with 1 <= m < 2; 7 = 1.75 * 2^2
  int k = static_cast<int>(bits >> 23) - 127 - 2 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  if (k < FP4_MIN_EXP) k = FP4_MIN_EXP;      // zeros and subnormals among them
  if (k > FP4_MAX_EXP) k = FP4_MAX_EXP;
  return k + 127;
}
__device__ __forceinline__ float fp4_factor(int byte) {   // 2^(byte - 127) for the bytes 2 .. 252
  return __uint_as_float(static_cast<uint32_t>(byte) << 23);
}
__device__ __forceinline__ float fp4_inverse(int byte) {  // 2^(127 - byte) for the bytes 2 .. 252
  return __uint_as_float(static_cast<uint32_t>(254 - byte) << 23);
}

// The code nearest to `y` (an element over its group's factor).  NaN gives code 0: its group's factor says so.
__device__ __forceinline__ uint32_t fp4_code(float y) {
  const float a = fabsf(y);
  const uint32_t size = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.f);
  return size | (__float_as_uint(y) >> 28 & 8u);
}

// The number a code stands for, without its group's factor.
__device__ __forceinline__ float fp4_level(uint32_t code) {
  const uint32_t size = code & 7u;
  // 0, 0.5, then 2^e * (1 or 1.5): the float with exponent 127 + e and the mantissa's top bit
  const uint32_t bits = size < 2 ? size * 0x3f000000u : (126u + (size >> 1)) << 23 | (size & 1u) << 22;
  return __uint_as_float(bits | (code & 8u) << 28);
}
// The value of a code in a group with this factor byte.
__device__ __forceinline__ float fp4_value(uint32_t code, int factor) {
  // a code times a power of two: exact, also as a bfloat16
  return factor == FP4_NAN ? __uint_as_float(0x7fc00000u) : fp4_level(code) * fp4_factor(factor);
}

// Two codes (byte BYTE of `word`, the lower half first) times a factor, as two bfloat16.  The instruction takes
// the exponent field of its float factor and looks at nothing else of it, so that a factor byte only has to be
// shifted to bits 23 to 30, whatever lies beside it; 255 gives two NaN.
#ifndef SE_FP4_PAIR
#define SE_FP4_PAIR(word, factor_bits, BYTE) \
  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, __uint_as_float(factor_bits), BYTE))
#endif
template <int BYTE>
__device__ __forceinline__ uint32_t fp4_factor_bits(uint32_t word) {   // byte BYTE of `word` as a float's exponent field
  return BYTE < 3 ? word << (23 - 8 * (BYTE < 3 ? BYTE : 0)) : word >> 1;
}
// eight codes (a word) under one factor: an operand's eight bfloat16
__device__ __forceinline__ uint4 fp4_eight(uint32_t word, uint32_t factor_bits) {
  uint4 r;
  r.x = SE_FP4_PAIR(word, factor_bits, 0);
  r.y = SE_FP4_PAIR(word, factor_bits, 1);
  r.z = SE_FP4_PAIR(word, factor_bits, 2);
  r.w = SE_FP4_PAIR(word, factor_bits, 3);
  return r;
}
