// Rows held in registers by a wave or by a workgroup: sums and maxima over a row in a fixed
// order, and eight values rounded to their type.
#pragma once

#include <type_traits>

#include "hmoe_common.h"
#include "quant_e4m3.h"

namespace hmoe {

// v + v of the lane the DPP control CTRL names, in the rows ROW_MASK enables.
template <int CTRL, int ROW_MASK = 0xF>
__device__ __forceinline__ float dpp_fadd(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROW_MASK, 0xF, false));
}
// Wave-wide, returned in every lane; the moves are those of wave_max_f32.
__device__ __forceinline__ float wave_sum_f32(float v) {
  v = dpp_fadd<0xB1>(v);
  v = dpp_fadd<0x4E>(v);
  v = dpp_fadd<0x141>(v);
  v = dpp_fadd<0x140>(v);
  v = dpp_fadd<0x142, 0xA>(v);
  v = dpp_fadd<0x143, 0xC>(v);
  return lane_bcast(v, 63);
}

// Over the NT threads (64, or the whole workgroup) that hold a row, in every thread of
// them.  `part` (NT / 64 words of LDS) is free again after the next barrier but one.
template <int NT>
__device__ __forceinline__ float row_sum(float v, float* part) {
  v = wave_sum_f32(v);
  if constexpr (NT > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) v += part[w];
  }
  return v;
}
template <int NT>
__device__ __forceinline__ int32_t row_max(int32_t v, int32_t* part) {
  v = wave_max_i32(v);
  if constexpr (NT > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) v = part[w] > v ? part[w] : v;
  }
  return v;
}

// Eight values stored in their type (16-byte aligned), and what that type keeps of them.
__device__ __forceinline__ void round_store8(float* o, const float (&v)[8]) {
  *reinterpret_cast<f32x4*>(o) = f32x4{v[0], v[1], v[2], v[3]};
  *reinterpret_cast<f32x4*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void round_store8(uint16_t* o, float (&v)[8]) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{v[2 * i], v[2 * i + 1]}, bf16x2_t));
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  *reinterpret_cast<u32x4*>(o) = w;
}

// Eight values of a bf16 (dtype HMOE_BF16) or float32 array.
__device__ __forceinline__ void load8(const void* p, int64_t at, bool bf16, float (&v)[8]) {
  if (bf16) {  // uniform
    Chunk8<uint16_t> c;
    c.load(static_cast<const uint16_t*>(p) + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c.get(i);
  } else {
    Chunk8<float> c;
    c.load(static_cast<const float*>(p) + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c.get(i);
  }
}

// How a row of `cols` values is held: NT threads and C chunks of eight values a thread, with
// which `f` is called.  A wave a row where there are rows enough to fill the chip with waves
// and rows are short enough (max_wave_cols): 100000 rows of 256 values are normed in 68 us by
// waves, 142 by workgroups, 30000 of 1024 in 61 and 70, 16384 of 2048 in the same time.  (The norm's
// gradients of 1000 rows of 8200 bf16 values take 27 us with two chunks a thread of 1024, 101 with
// four, which a thread's 128 registers do not hold.)
constexpr int kMaxRowCols = 32768;
constexpr int64_t kWaveRows = 2048;
template <int N>
using Int = std::integral_constant<int, N>;
template <typename F>
void with_row_form(int64_t rows, int cols, int max_wave_cols, F f) {
  const int chunks = cols / 8;
  const bool wave = rows >= kWaveRows && cols <= max_wave_cols;
  if (wave && chunks <= 64 * 2) f(Int<64>{}, Int<2>{});
  else if (wave && chunks <= 64 * 4) f(Int<64>{}, Int<4>{});
  else if (chunks <= 256) f(Int<256>{}, Int<1>{});
  else if (chunks <= 256 * 2) f(Int<256>{}, Int<2>{});
  else if (chunks <= 256 * 4) f(Int<256>{}, Int<4>{});
  else if (chunks <= 1024 * 2) f(Int<1024>{}, Int<2>{});
  else f(Int<1024>{}, Int<4>{});
}

// Workgroups of a launch over rows (a launch has fewer than 2^32 threads along x).
inline unsigned row_grid(int64_t rows, int rows_per_group) {
  const int64_t g = ceil_div(rows, rows_per_group);
  return static_cast<unsigned>(g < (1 << 20) ? g : (1 << 20));
}

}  // namespace hmoe
