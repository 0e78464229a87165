// MXFP4: 32 consecutive values of a row share a power-of-two scale, an E8M0
// byte E standing for 2^(E - 127), and each value is a 4-bit e2m1 code (sign,
// two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6).
//
// The scale is the smallest power of two at which the block's largest value
// rounds to 6 or less: with amax = m 2^a, 1 <= m < 2, that is 2^(a - 2) where m <
// 1.75 (then amax is below 7 scale units, which rounds to 6 at most) and 2^(a - 1)
// above.  (Always 2^(a - 2), as in the conversion that the OCP Microscaling Formats
// specification describes, would cut values of 7 to 8 units to 6.)  Adding a
// quarter to the mantissa field carries into the exponent exactly where m >= 1.75.
// Scaling by a power of two is exact, so a code is one rounding (nearest, ties to
// the even code) of the value.  A block with a value that is not finite gets E =
// 255, the format's NaN, and zero codes.
#pragma once

#include <initializer_list>

#include "hmoe_common.h"

namespace hmoe {

constexpr int kMxBlock = 32;

// Codes and values are read and written 16 bytes at a time, exponents by words.
inline bool aligned_to(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
#define HMOE_REQUIRE_ALIGNED(what, bytes, ...)                                                \
  do {                                                                                        \
    for (const void* p_ : std::initializer_list<const void*>{__VA_ARGS__})                    \
      HMOE_REQUIRE(::hmoe::aligned_to(p_, bytes), "%s: an operand is not %d-byte aligned", (what), (bytes)); \
  } while (0)

// E from the largest of the block's |v| as float32 bits (as integers they order
// like the values, infinities and NaNs on top).
__device__ __forceinline__ uint32_t mxfp4_exponent(uint32_t amax_bits) {
  const uint32_t up = (amax_bits + 0x200000u) >> 23;
  const uint32_t e = up > 2u ? up - 2u : 0u;
  return amax_bits >= 0x7f800000u ? 255u : e;
}

// 2^(E - 127), NaN at 255 (2^-127 is below float32's normal numbers).
__device__ __forceinline__ float mxfp4_scale(uint32_t e) {
  return __uint_as_float(e == 0u ? 0x00400000u : e == 255u ? 0x7fc00000u : e << 23);
}

// Codes of eight values of a block with exponent e, value i in bits 4 i .. 4 i + 3.  (The
// conversion divides by its scale operand, of which it takes the exponent field alone.)
__device__ __forceinline__ uint32_t mxfp4_codes8(const float (&v)[8], uint32_t e) {
  const float scale = __uint_as_float(e << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
  // (the codes of infinities and NaNs are left open)
  return e != 255u ? w : 0u;
}

__device__ __forceinline__ uint32_t umax32(uint32_t a, uint32_t b) { return a > b ? a : b; }

// Eight values of a row (chunk c of it) to a word of codes, and the block's exponent.  Four
// neighbouring lanes hold a block.
template <typename Values>
__device__ __forceinline__ void quant_chunk_mxfp4(const Values& x, int64_t c, uint8_t* q, uint8_t* exps) {
  float v[8];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = x.get(i);
    amax = umax32(amax, __float_as_uint(v[i]) & 0x7fffffffu);
  }
  amax = umax32(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 1)));
  amax = umax32(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 2)));
  const uint32_t e = mxfp4_exponent(amax);
  reinterpret_cast<uint32_t*>(q)[c] = mxfp4_codes8(v, e);
  if ((c & 3) == 0) exps[c >> 2] = static_cast<uint8_t>(e);
}

// The eight values of a word of codes.
__device__ __forceinline__ void mxfp4_values8(uint32_t w, float scale, float (&v)[8]) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
  const f32x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
  const f32x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2);
  const f32x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
  v[0] = a[0] * scale;
  v[1] = a[1] * scale;
  v[2] = b[0] * scale;
  v[3] = b[1] * scale;
  v[4] = c[0] * scale;
  v[5] = c[1] * scale;
  v[6] = d[0] * scale;
  v[7] = d[1] * scale;
}

}  // namespace hmoe
