// int8 rows and operands: quantising, reading back (e4m3 rows too), and packing the expert
// masters for the grouped products (quant_i8.h has the rule).  Bound by memory: a row is
// read once and held in registers.
#include "quant_i8.h"
#include "quant_mxfp4.h"
#include "rows.h"

namespace hmoe {
namespace {

// NT threads a row, C chunks of eight values each.  Rows past offsets[n_experts] (where
// offsets are given) are not read: their codes are left, their scale is 1.  131072 x 1024 in bf16:
// 62 us for 403 MB, 16384 x 2048: 19 us for 101 MB.
template <typename TI, int NT, int C>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void quantize_rows_i8_kernel(
    const TI* __restrict__ a, int64_t rows, int cols, const int32_t* __restrict__ offsets, int n_experts,
    int8_t* __restrict__ q, float* __restrict__ scale) {
  constexpr int kThreads = NT < 256 ? 256 : NT;
  __shared__ int32_t part[2][NT / 64];
  const int t = threadIdx.x % NT;
  const int chunks = cols / 8;
  const int64_t live = offsets != nullptr ? offsets[n_experts] : rows;
  int parity = 0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / NT) + threadIdx.x / NT; row < rows;
       row += static_cast<int64_t>(gridDim.x) * (kThreads / NT), parity ^= 1) {
    if (row >= live) {  // uniform over a row's threads
      if (t == 0) scale[row] = 1.0f;
      continue;
    }
    const int64_t r0 = row * cols;
    Chunk8<TI> x[C];
#pragma unroll
    for (int u = 0; u < C; ++u) {
      const int c = u * NT + t;
      x[u].zero();
      if (c < chunks) x[u].load_nt(a + r0 + c * 8);
    }
    int32_t most = 0;
    float v[C][8];
#pragma unroll
    for (int u = 0; u < C; ++u) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u][i] = x[u].get(i);
      most = amax8_bits(v[u], most);
    }
    const I8Scale s = i8_scale(row_max<NT>(most, part[parity]));
    if (t == 0) scale[row] = s.scale;
#pragma unroll
    for (int u = 0; u < C; ++u) {
      const int c = u * NT + t;
      if (c < chunks) *reinterpret_cast<uint2*>(q + r0 + c * 8) = i8_codes8(v[u], s);
    }
  }
}

// Eight codes to their values.
__device__ __forceinline__ void values8(const int8_t* p, float (&v)[8]) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = static_cast<float>(static_cast<int32_t>(w.x << (24 - 8 * i)) >> 24);
    v[4 + i] = static_cast<float>(static_cast<int32_t>(w.y << (24 - 8 * i)) >> 24);
  }
}
struct E4m3 {
  uint8_t code;
};
__device__ __forceinline__ void values8(const E4m3* p, float (&v)[8]) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w.x), false);
  const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w.x), true);
  const auto c = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w.y), false);
  const auto d = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w.y), true);
  v[0] = a[0];
  v[1] = a[1];
  v[2] = b[0];
  v[3] = b[1];
  v[4] = c[0];
  v[5] = c[1];
  v[6] = d[0];
  v[7] = d[1];
}

// A wave a row: 16384 x 2048 to bf16 in 16 us, 101 MB.
template <typename TQ, typename TO>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(const TQ* __restrict__ q, const float* __restrict__ scale,
                                                              int64_t rows, int cols, TO* __restrict__ out) {
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); row < rows;
       row += static_cast<int64_t>(gridDim.x) * 4) {
    const float s = scale[row];
    for (int c = threadIdx.x & 63; c < cols / 8; c += 64) {
      float v[8];
      values8(q + row * cols + c * 8, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= s;
      round_store8(out + row * cols + c * 8, v);
    }
  }
}

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(uint16_t v) { return bf16_bits_to_f32(v); }

// 32 columns of a master src[e][K][C] a workgroup: their largest values over all of K, then
// their codes.  Lane 32 h + r takes column r of 16 consecutive values of K, which are the 16
// bytes that the matrix instruction's lane holds: a wave writes runs of 1 KB.  The second
// pass finds part of the columns in the caches.  GATE_UP: grid.z counts gate, then up, of each
// expert.  64 experts, D 2048, F 1024, float32 masters: 443 us gate/up (1.34 GB if each master
// is read once), 186 down; in bf16, whose runs along a row are 64 bytes, 349 and 183.  It runs
// once for an update of the weights.
constexpr int kPackWaves = 8;
template <typename TW, bool GATE_UP>
__global__ __launch_bounds__(64 * kPackWaves) void pack_i8_kernel(const TW* __restrict__ src0,
                                                                  const TW* __restrict__ src1, int kdim, int cols,
                                                                  int8_t* __restrict__ dst,
                                                                  float* __restrict__ scales) {
  __shared__ int32_t part[kPackWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int half = lane >> 5, r = lane & 31;
  const int e = GATE_UP ? blockIdx.z >> 1 : blockIdx.z;
  const int which = GATE_UP ? blockIdx.z & 1 : 0;
  const int rows = GATE_UP ? 2 * cols : cols;
  const int c0 = blockIdx.x * 32;
  const TW* src = (which ? src1 : src0) + static_cast<int64_t>(e) * kdim * cols + c0 + r;
  const int blocks = kdim / 32;
  int32_t most = 0;
  const auto load = [&](int kb, float (&v)[16]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = widen(src[static_cast<int64_t>(kb * 32 + half * 16 + i) * cols]);
  };
  for (int kb = wave; kb < blocks; kb += kPackWaves) {
    float v[16];
    load(kb, v);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int32_t b = __float_as_int(v[i]) & 0x7fffffff;
      most = b > most ? b : most;
    }
  }
  part[wave][lane] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kPackWaves; ++w) {
    most = part[w][r] > most ? part[w][r] : most;
    most = part[w][32 + r] > most ? part[w][32 + r] : most;
  }
  const I8Scale s = i8_scale(most);
  // operand row of column c0: blocks of 32 gate and 32 up columns alternate
  const int p0 = GATE_UP ? c0 * 2 + which * 32 : c0;
  if (wave == 0 && half == 0) scales[static_cast<int64_t>(e) * rows + p0 + r] = s.scale;
  int8_t* out = dst + (static_cast<int64_t>(e) * (rows / 32) + p0 / 32) * blocks * 1024 + lane * 16;
  for (int kb = wave; kb < blocks; kb += kPackWaves) {
    float v[16];
    load(kb, v);
    u32x4 w;
#pragma unroll
    for (int g = 0; g < 4; ++g)
      w[g] = pack4_u8(i8_code(v[4 * g], s), i8_code(v[4 * g + 1], s), i8_code(v[4 * g + 2], s),
                      i8_code(v[4 * g + 3], s));
    *reinterpret_cast<u32x4*>(out + static_cast<int64_t>(kb) * 1024) = w;
  }
}

int check_operand(const char* what, int n_experts, int d_model, int d_ff) {
  HMOE_REQUIRE(n_experts >= 1 && n_experts <= 1024, "%s: n_experts must be in [1, 1024] (got %d)", what, n_experts);
  HMOE_REQUIRE_CODE(d_model >= 128 && d_model % 128 == 0 && d_model <= kMaxRowCols, HMOE_ERR_UNSUPPORTED,
                    "%s: d_model must be a multiple of 128 up to %d (got %d)", what, kMaxRowCols, d_model);
  HMOE_REQUIRE_CODE(d_ff >= 128 && d_ff % 128 == 0 && d_ff <= kMaxRowCols, HMOE_ERR_UNSUPPORTED,
                    "%s: d_ff must be a multiple of 128 up to %d (got %d)", what, kMaxRowCols, d_ff);
  return HMOE_OK;
}

int pack_i8(const char* what, const void* w0, const void* w1, int w_dtype, int n_experts, int kdim, int cols,
            int8_t* packed, float* scales, hipStream_t s) {
  const bool gate_up = w1 != nullptr;
  const dim3 grid(cols / 32, 1, gate_up ? 2 * n_experts : n_experts);
#define HMOE_LAUNCH_PACK8(TW, GU)                                                                 \
  hipLaunchKernelGGL((pack_i8_kernel<TW, GU>), grid, dim3(64 * kPackWaves), 0, s,                 \
                     static_cast<const TW*>(w0), static_cast<const TW*>(w1), kdim, cols, packed, scales)
  if (w_dtype == HMOE_F32 && gate_up) HMOE_LAUNCH_PACK8(float, true);
  else if (w_dtype == HMOE_F32) HMOE_LAUNCH_PACK8(float, false);
  else if (gate_up) HMOE_LAUNCH_PACK8(uint16_t, true);
  else HMOE_LAUNCH_PACK8(uint16_t, false);
#undef HMOE_LAUNCH_PACK8
  return check_launch(what);
}

template <typename TQ>
int dequantize_rows(const char* what, const void* q, const float* scale, int64_t rows, int cols, void* out,
                    int out_dtype, hmoe_stream_t stream) {
  HMOE_REQUIRE(rows >= 0 && rows <= (int64_t(1) << 40), "%s: rows must be in [0, 2^40]", what);
  HMOE_REQUIRE_CODE(cols >= 8 && cols % 8 == 0, HMOE_ERR_UNSUPPORTED, "%s: cols must be a multiple of 8 (got %d)",
                    what, cols);
  HMOE_REQUIRE(out_dtype == HMOE_F32 || out_dtype == HMOE_BF16, "%s: out dtype must be F32 or BF16", what);
  if (rows == 0) return HMOE_OK;
  HMOE_REQUIRE(q && scale && out, "%s: null pointer argument", what);
  HMOE_REQUIRE_ALIGNED(what, 16, out);
  HMOE_REQUIRE_ALIGNED(what, 8, q);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(row_grid(rows, 4));
  if (out_dtype == HMOE_F32)
    hipLaunchKernelGGL((dequantize_rows_kernel<TQ, float>), grid, dim3(256), 0, s, static_cast<const TQ*>(q), scale,
                       rows, cols, static_cast<float*>(out));
  else
    hipLaunchKernelGGL((dequantize_rows_kernel<TQ, uint16_t>), grid, dim3(256), 0, s, static_cast<const TQ*>(q), scale,
                       rows, cols, static_cast<uint16_t*>(out));
  return check_launch(what);
}

}  // namespace
}  // namespace hmoe

extern "C" int hmoe_quantize_rows_i8(const void* a, int a_dtype, int64_t rows, int cols, const int32_t* offsets,
                                     int n_experts, int8_t* q, float* scale, hmoe_stream_t stream) {
  using namespace hmoe;
  const char* what = "quantize_rows_i8";
  HMOE_REQUIRE(rows >= 0 && rows <= (int64_t(1) << 40), "%s: rows must be in [0, 2^40]", what);
  HMOE_REQUIRE_CODE(cols >= 8 && cols % 8 == 0 && cols <= kMaxRowCols, HMOE_ERR_UNSUPPORTED,
                    "%s: cols must be a multiple of 8 up to %d (got %d)", what, kMaxRowCols, cols);
  HMOE_REQUIRE(a_dtype == HMOE_F32 || a_dtype == HMOE_BF16, "%s: a dtype must be F32 or BF16", what);
  HMOE_REQUIRE(offsets == nullptr || (n_experts >= 0 && n_experts <= 1024), "%s: n_experts must be in [0, 1024]", what);
  if (rows == 0) return HMOE_OK;
  HMOE_REQUIRE(a && q && scale, "%s: null pointer argument", what);
  HMOE_REQUIRE_ALIGNED(what, 16, a);
  HMOE_REQUIRE_ALIGNED(what, 8, q);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto launch = [&](auto nt, auto c) {
    constexpr int kNt = decltype(nt)::value, kC = decltype(c)::value;
    constexpr int kThreads = kNt < 256 ? 256 : kNt;
    const dim3 grid(row_grid(rows, kThreads / kNt));
    if (a_dtype == HMOE_BF16)
      hipLaunchKernelGGL((quantize_rows_i8_kernel<uint16_t, kNt, kC>), grid, dim3(kThreads), 0, s,
                         static_cast<const uint16_t*>(a), rows, cols, offsets, n_experts, q, scale);
    else
      hipLaunchKernelGGL((quantize_rows_i8_kernel<float, kNt, kC>), grid, dim3(kThreads), 0, s,
                         static_cast<const float*>(a), rows, cols, offsets, n_experts, q, scale);
  };
  with_row_form(rows, cols, 2048, launch);
  return check_launch("hmoe_quantize_rows_i8");
}

extern "C" int hmoe_dequantize_rows_i8(const int8_t* q, const float* scale, int64_t rows, int cols, void* out,
                                       int out_dtype, hmoe_stream_t stream) {
  return hmoe::dequantize_rows<int8_t>("dequantize_rows_i8", q, scale, rows, cols, out, out_dtype, stream);
}

extern "C" int hmoe_dequantize_rows_fp8(const uint8_t* q, const float* scale, int64_t rows, int cols, void* out,
                                        int out_dtype, hmoe_stream_t stream) {
  return hmoe::dequantize_rows<hmoe::E4m3>("dequantize_rows_fp8", q, scale, rows, cols, out, out_dtype, stream);
}

extern "C" size_t hmoe_packed_i8_gate_up_bytes(int n_experts, int d_model, int d_ff) {
  if (n_experts <= 0 || d_model <= 0 || d_ff <= 0) return 0;
  return static_cast<size_t>(n_experts) * 2 * d_ff * d_model;
}

extern "C" size_t hmoe_packed_i8_down_bytes(int n_experts, int d_ff, int d_model) {
  if (n_experts <= 0 || d_model <= 0 || d_ff <= 0) return 0;
  return static_cast<size_t>(n_experts) * d_ff * d_model;
}

extern "C" int hmoe_pack_i8_gate_up(const void* w_gate, const void* w_up, int w_dtype, int n_experts, int d_model,
                                    int d_ff, int8_t* packed, float* scales, hmoe_stream_t stream) {
  using namespace hmoe;
  const char* what = "pack_i8_gate_up";
  if (int rc = check_operand(what, n_experts, d_model, d_ff)) return rc;
  HMOE_REQUIRE(w_dtype == HMOE_F32 || w_dtype == HMOE_BF16, "%s: weight dtype must be F32 or BF16", what);
  HMOE_REQUIRE(w_gate && w_up && packed && scales, "%s: null pointer argument", what);
  HMOE_REQUIRE_ALIGNED(what, 16, packed);
  return pack_i8("hmoe_pack_i8_gate_up", w_gate, w_up, w_dtype, n_experts, d_model, d_ff, packed, scales,
                 static_cast<hipStream_t>(stream));
}

extern "C" int hmoe_pack_i8_down(const void* w_down, int w_dtype, int n_experts, int d_ff, int d_model,
                                 int8_t* packed, float* scales, hmoe_stream_t stream) {
  using namespace hmoe;
  const char* what = "pack_i8_down";
  if (int rc = check_operand(what, n_experts, d_model, d_ff)) return rc;
  HMOE_REQUIRE(w_dtype == HMOE_F32 || w_dtype == HMOE_BF16, "%s: weight dtype must be F32 or BF16", what);
  HMOE_REQUIRE(w_down && packed && scales, "%s: null pointer argument", what);
  HMOE_REQUIRE_ALIGNED(what, 16, packed);
  return pack_i8("hmoe_pack_i8_down", w_down, nullptr, w_dtype, n_experts, d_ff, d_model, packed, scales,
                 static_cast<hipStream_t>(stream));
}
