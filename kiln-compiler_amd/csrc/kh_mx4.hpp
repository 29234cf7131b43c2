// kh_mx4.hpp - keys and values in 4 bits (KH_TYPE_MX4): 32 adjacent dimensions
// of a token share a power of two 2^(e - 127), an element is a sign and one of
// 0, .5, 1, 1.5, 2, 3, 4, 6 times it.
//
// The format is what gfx950 converts in one instruction a pair (and multiplies
// in its scaled matrix instructions), and every value it holds is a bf16 one:
// attention over it is attention over a bf16 cache that takes 17/64 of the
// bytes. e is the smallest for which the block's largest rounds to 6 at most
// (below 7 steps of it), at least 2 and at most 252 so that no value is
// subnormal or past fp32 (6 2^125 is the largest); elements go to the nearest,
// ties to the even code. A block with an element that is not
// finite has e = 255 and is NaN.
//
// A page of a head is page_size tokens of dim / 2 code bytes, then as many of
// dim / 32 scale bytes. Keys lie token by token: a lane of the first product
// reads 32 (or 16, 64) adjacent dimensions of one key. Values lie 16 tokens
// together, 4 of them x 8 dimensions in 16 bytes, which is what a lane of the
// second product reads of them; a token's scales likewise, 4 tokens in 4 bytes.
#pragma once

#include <cmath>
#include <cstdint>
#include <cstring>

#include "kh_common.hpp"

namespace kh {

constexpr int kMxBlock = 32;
constexpr uint32_t kMxMost = 252;   // the largest scale byte of numbers; 255 is NaN's, the two between nobody's

// Byte offsets inside a page of a head, of token t's element d (its low half
// where d is even) and of its block's scale byte.
__host__ __device__ inline int mx_page_bytes(int page_size, int dim) { return page_size * (dim / 2 + dim / kMxBlock); }
__host__ __device__ inline int mx_key_code(int t, int d, int dim) { return t * (dim / 2) + d / 2; }
__host__ __device__ inline int mx_key_scale(int t, int d, int dim, int page_size) {
  return page_size * (dim / 2) + t * (dim / kMxBlock) + d / kMxBlock;
}
__host__ __device__ inline int mx_value_code(int t, int d, int dim) {
  return (t >> 4) * 8 * dim + (((t & 15) >> 2) * (dim / 8) + d / 8) * 16 + (t & 3) * 4 + (d & 7) / 2;
}
__host__ __device__ inline int mx_value_scale(int t, int d, int dim, int page_size) {
  return page_size * (dim / 2) + (t >> 4) * (dim / 2) + (((t & 15) >> 2) * (dim / kMxBlock) + d / kMxBlock) * 4 + (t & 3);
}

// The scale byte of a block whose largest |x| has these bits (NaN and inf are
// the largest bits of all).
__host__ __device__ inline uint32_t mx_scale_of(uint32_t most) {
  if (most >= 0x7f800000u) return 255u;
  const int e = (int)(most >> 23) - 2 + ((most & 0x7fffffu) >= 0x600000u ? 1 : 0);
  return e < 2 ? 2u : e > (int)kMxMost ? kMxMost : (uint32_t)e;
}

// -- on the CPU -------------------------------------------------------------------

inline float mx_value(uint32_t code, uint32_t e) {
  static const float level[8] = {0.0f, 0.5f, 1.0f, 1.5f, 2.0f, 3.0f, 4.0f, 6.0f};
  if (e > kMxMost) return std::nanf("");
  const float x = std::ldexp(level[code & 7], (int)e - 127);
  return code & 8 ? -x : x;
}

inline uint32_t mx_bits(float x) {
  uint32_t u;
  std::memcpy(&u, &x, 4);
  return u;
}

inline uint32_t mx_code(float x, uint32_t e) {
  if (e == 255) return 0;
  const double y = std::ldexp(std::fabs((double)x), 127 - (int)e);
  // the middles between levels; a tie goes to the even code
  uint32_t code = (y > 0.25) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0);
  return code | (mx_bits(x) >> 31) << 3;
}

// x[0 .. 32) as the cache holds it
inline void mx_round(float *x) {
  uint32_t most = 0;
  for (int i = 0; i < kMxBlock; ++i) most = std::max(most, mx_bits(x[i]) & 0x7fffffffu);
  const uint32_t e = mx_scale_of(most);
  for (int i = 0; i < kMxBlock; ++i) x[i] = mx_value(mx_code(x[i], e), e);
}

// -- on the device -----------------------------------------------------------------

typedef __bf16 mx_bf16x2 __attribute__((ext_vector_type(2)));
typedef float mx_f32x2 __attribute__((ext_vector_type(2)));

// The power of two of a scale byte, or NaN.
__device__ __forceinline__ float mx_scale(uint32_t e) { return __uint_as_float(e > kMxMost ? 0x7fc00000u : e << 23); }

// ... left to the conversions, which take an exponent of 255 for NaN. (253 and 254,
// which no writer makes and whose blocks are not defined, they take for 2^126 and
// 2^127: telling them apart would cost paged_mx4_kernel 1.2% of its time, 43.6
// to 44.1 us for 32 ragged sequences.)
__device__ __forceinline__ float mx_scale_raw(uint32_t e) { return __uint_as_float(e << 23); }

// Codes 2 i and 2 i + 1 of a word as a pair of bf16, exact.
template <int I>
__device__ __forceinline__ uint32_t mx_pair(uint32_t word, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, I));
}

// 8 codes of a word as floats.
__device__ __forceinline__ void mx_unpack(uint32_t word, float scale, float (&x)[8]) {
  const mx_f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 1),
                 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 3);
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y, x[4] = c.x, x[5] = c.y, x[6] = d.x, x[7] = d.y;
}

// Largest bits of |x|.
template <int N>
__device__ __forceinline__ uint32_t mx_most(const float (&x)[N]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  return m;
}

// The largest of a quad of lanes.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
}

// 8 values as codes under scale byte e.
__device__ __forceinline__ uint32_t mx_pack(const float (&x)[8], uint32_t e) {
  const float scale = __uint_as_float((e == 255u ? 127u : e) << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
  return e == 255u ? 0u : w;
}

}  // namespace kh
