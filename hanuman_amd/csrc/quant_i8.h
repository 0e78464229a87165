// int8 rows: a row's scale is its largest |v| over 127, a code v (127 / largest) rounded to
// nearest even, both quotients correctly rounded float32; a row of zeros has scale 1.  In
// float32 the product is off by 2^-23 of itself.  A bfloat16 row's codes are nevertheless the
// nearest to the exact quotients: with v = a 2^i, largest = b 2^j (a, b < 256) a quotient is a
// half where 254 a = (2 k + 1) b 2^n, integers below 2^16, which differ by a part in 2^16 if
// they do.  A row with a value that is not finite has zero codes and a scale that is not finite:
// it reads back as NaN, and so does every product with it.
#pragma once

#include "hmoe_common.h"

namespace hmoe {

constexpr float kI8Max = 127.0f;

// Largest |v| as float32 bits (as integers they order like the values, infinities and NaNs
// on top) of the values v[0..7] and of `most`.
__device__ __forceinline__ int32_t amax8_bits(const float (&v)[8], int32_t most) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int32_t b = __float_as_int(v[i]) & 0x7fffffff;
    most = b > most ? b : most;
  }
  return most;
}

// v is multiplied by `up`, then by `inv`: 127 / amax overflows below 2^-121, so the rows of
// such values are first taken up by 2^64.
struct I8Scale {
  float scale, up, inv;
};
__device__ __forceinline__ I8Scale i8_scale(int32_t amax_bits) {
#pragma clang fp contract(off)
  const float amax = __int_as_float(amax_bits);
  I8Scale s;
  s.up = amax < 0x1p-64f ? 0x1p64f : 1.0f;
  s.scale = amax == 0.0f ? 1.0f : amax / kI8Max;
  // (infinity: 0; NaN: NaN.  A product of either with what is not finite is NaN, code 0)
  s.inv = amax == 0.0f ? 0.0f : kI8Max / (amax * s.up);
  return s;
}
__device__ __forceinline__ uint32_t i8_code(float v, const I8Scale& s) {
#pragma clang fp contract(off)
  return static_cast<uint32_t>(static_cast<int32_t>(__builtin_rintf(v * s.up * s.inv)));
}
__device__ __forceinline__ uint32_t pack4_u8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return (a & 0xffu) | ((b & 0xffu) << 8) | ((c & 0xffu) << 16) | (d << 24);
}
__device__ __forceinline__ uint2 i8_codes8(const float (&v)[8], const I8Scale& s) {
  uint32_t q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = i8_code(v[i], s);
  return uint2{pack4_u8(q[0], q[1], q[2], q[3]), pack4_u8(q[4], q[5], q[6], q[7])};
}

}  // namespace hmoe
