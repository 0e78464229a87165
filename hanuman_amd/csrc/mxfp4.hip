// MXFP4 rows and operands: quantising, reading back, and packing the expert
// masters for the grouped products (quant_mxfp4.h has the format).  All of it is
// bound by memory: no value is looked at twice.
#include "quant_mxfp4.h"
#include "quant_e4m3.h"

namespace hmoe {
namespace {

// Rows are whole blocks, so a matrix is one run of them.  A lane takes eight
// values and four neighbours a block.
template <typename TI>
__global__ __launch_bounds__(256) void quantize_rows_mxfp4_kernel(const TI* __restrict__ a,
                                                                  int64_t chunks,
                                                                  uint8_t* __restrict__ q,
                                                                  uint8_t* __restrict__ exps) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; c < chunks; c += stride) {
    Chunk8<TI> x;
    x.load_nt(a + c * 8);
    quant_chunk_mxfp4(x, c, q, exps);  // (chunks is a multiple of 4: a block's lanes are here together)
  }
}

// Eight values of a row.  PAST: past the caches, for matrices that they cannot hold.
template <bool PAST, typename V>
__device__ __forceinline__ void store16(V* o, V v) {
  if (PAST) __builtin_nontemporal_store(v, o);
  else *o = v;
}
template <bool PAST>
__device__ __forceinline__ void store8(float* o, const float (&v)[8]) {
  store16<PAST>(reinterpret_cast<f32x4*>(o), f32x4{v[0], v[1], v[2], v[3]});
  store16<PAST>(reinterpret_cast<f32x4*>(o + 4), f32x4{v[4], v[5], v[6], v[7]});
}
// (the values have two significant bits: the upper half of the float32 is all of them)
template <bool PAST>
__device__ __forceinline__ void store8(uint16_t* o, const float (&v)[8]) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = (__float_as_uint(v[2 * i]) >> 16) | (__float_as_uint(v[2 * i + 1]) & 0xffff0000u);
  store16<PAST>(reinterpret_cast<u32x4*>(o), w);
}

// Written values that are more than the L2s (8 x 4 MB) go past them: 134 M values to
// bf16 (268 MB) take 65 us through them and 47 past them, 33 M 13.6 and 11.2.  Fewer are
// left to the caches, from which what follows reads them.
constexpr int64_t kCachedBytes = int64_t(32) << 20;

template <typename TO, bool PAST>
__global__ __launch_bounds__(256) void dequantize_rows_mxfp4_kernel(const uint8_t* __restrict__ q,
                                                                    const uint8_t* __restrict__ exps,
                                                                    int64_t chunks, TO* __restrict__ out) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; c < chunks; c += stride) {
    float v[8];
    mxfp4_values8(reinterpret_cast<const uint32_t*>(q)[c], mxfp4_scale(exps[c >> 2]), v);
    store8<PAST>(out + c * 8, v);
  }
}

// A packed operand's values row by row.  A workgroup takes 32 rows x 64 kUnpackBlocks
// columns, eight values a thread and block of 1 KB, so that eight threads write a run of
// 128 (bf16) or 256 bytes.  Bound by memory: 268 M values to bf16 (0.68 GB moved) in
// 145 us; found by dividing a flat index it took 232 us, most of it the divisions.
constexpr int kUnpackBlocks = 4;
template <typename TO, bool PAST>
__global__ __launch_bounds__(256) void unpack_mxfp4_kernel(const uint8_t* __restrict__ packed,
                                                           const uint8_t* __restrict__ exps, int rows, int cols,
                                                           TO* __restrict__ out) {
  const int row = threadIdx.x >> 3, k8 = threadIdx.x & 7;  // columns 8 k8 .. + 8 of a block
  const int64_t row32 = blockIdx.x;                        // of all experts'
  const int64_t n = row32 / (rows / 32);
  const int p = static_cast<int>(row32 - n * (rows / 32)) * 32 + row;
  const int blocks = cols / 64, first = blockIdx.y * kUnpackBlocks;
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(packed) + row32 * blocks * 256 +
                          ((k8 >> 2) * 32 + row) * 4 + (k8 & 3);
  const uint8_t* ex = exps + n * (cols / 32) * rows + p * 4 + (k8 >> 2);
  TO* o = out + (row32 * 32 + row) * cols + k8 * 8;
  uint32_t w[kUnpackBlocks];
  uint32_t e[kUnpackBlocks];
#pragma unroll
  for (int j = 0; j < kUnpackBlocks; ++j) {
    const int b = first + j;
    if (b < blocks) {
      w[j] = codes[static_cast<int64_t>(b) * 256];
      e[j] = ex[static_cast<int64_t>(b >> 1) * rows * 4 + (b & 1) * 2];
    }
  }
#pragma unroll
  for (int j = 0; j < kUnpackBlocks; ++j) {
    const int b = first + j;
    if (b < blocks) {
      float v[8];
      mxfp4_values8(w[j], mxfp4_scale(e[j]), v);
      store8<PAST>(o + b * 64, v);
    }
  }
}

// Two neighbouring columns of a master, which is read once (past the caches: 268 M
// float32 masters packed in 213 us, through them in 237).
__device__ __forceinline__ void load2(const float* p, float& a, float& b) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t v = __builtin_nontemporal_load(reinterpret_cast<const f32x2_t*>(p));
  a = v[0];
  b = v[1];
}
__device__ __forceinline__ void load2(const uint16_t* p, float& a, float& b) {
  const uint32_t v = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  a = __uint_as_float(v << 16);
  b = __uint_as_float(v & 0xffff0000u);
}

// One wave: 64 columns x 128 rows of a master src[e][K][C], which are 64 operand
// rows x 128 of the reduction.  Lane 32 h + i takes columns 2 i, 2 i + 1 of
// blocks h and 2 + h: its 32 values of a column are a block and, packed, the 16
// bytes that the matrix instruction's lane holds, so nothing moves between lanes
// but the exponents.  GATE_UP: grid.z counts gate, then up, of each expert.
template <typename TW, bool GATE_UP>
__global__ __launch_bounds__(256) void pack_mxfp4_kernel(const TW* __restrict__ src0,
                                                         const TW* __restrict__ src1, int kdim,
                                                         int cols, uint8_t* __restrict__ dst,
                                                         uint8_t* __restrict__ exps) {
  const int lane = threadIdx.x & 63;
  const int half = lane >> 5, i2 = (lane & 31) * 2;
  const int c0 = blockIdx.x * 64;
  const int kb = blockIdx.y * 4 + (threadIdx.x >> 6);  // 128 rows of the reduction
  if (kb * 128 >= kdim) return;
  const int e = GATE_UP ? blockIdx.z >> 1 : blockIdx.z;
  const int which = GATE_UP ? blockIdx.z & 1 : 0;
  const int rows = GATE_UP ? 2 * cols : cols;
  const TW* src = (which ? src1 : src0) + static_cast<int64_t>(e) * kdim * cols + c0 + i2;
  uint32_t ex[2] = {0, 0};  // this lane's columns' exponent words
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int k0 = kb * 128 + b * 64 + half * 32;
    float v[2][32];
    uint32_t amax[2] = {0, 0};
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      load2(src + static_cast<int64_t>(k0 + r) * cols, v[0][r], v[1][r]);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int r = 0; r < 32; ++r) amax[j] = umax32(amax[j], __float_as_uint(v[j][r]) & 0x7fffffffu);
      const uint32_t ee = mxfp4_exponent(amax[j]);
      u32x4 w;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float t[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) t[r] = v[j][g * 8 + r];
        w[g] = mxfp4_codes8(t, ee);
      }
      // column c of the master is operand row p
      const int c = c0 + i2 + j;
      const int p = GATE_UP ? (c >> 5) * 64 + which * 32 + (c & 31) : c;
      const int64_t frag = (static_cast<int64_t>(e) * (rows / 32) + p / 32) * (kdim / 64) + kb * 2 + b;
      *reinterpret_cast<u32x4*>(dst + (frag * 64 + half * 32 + (p & 31)) * 16) = w;
      ex[j] |= ee << (16 * b + 8 * half);
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t word = ex[j] | static_cast<uint32_t>(__shfl_xor(static_cast<int>(ex[j]), 32));
    const int c = c0 + i2 + j;
    const int p = GATE_UP ? (c >> 5) * 64 + which * 32 + (c & 31) : c;
    if (half == 0)
      *reinterpret_cast<uint32_t*>(exps + ((static_cast<int64_t>(e) * (kdim / 128) + kb) * rows + p) * 4) = word;
  }
}

unsigned chunk_grid(int64_t chunks) {
  const int64_t blocks = ceil_div(chunks, 256);
  return static_cast<unsigned>(blocks < 65536 ? blocks : 65536);
}

int pack_mxfp4(const char* what, const void* w0, const void* w1, int w_dtype, int n_experts, int kdim,
               int cols, uint8_t* packed, uint8_t* exps, hipStream_t s) {
  const bool gate_up = w1 != nullptr;
  const int z = gate_up ? 2 * n_experts : n_experts;
  HMOE_REQUIRE(ceil_div(kdim / 128, 4) <= 65535, "%s: reduction dimension too large", what);
  const dim3 grid(cols / 64, static_cast<unsigned>(ceil_div(kdim / 128, 4)), z);
#define HMOE_LAUNCH_PACK4(TW, GU)                                                              \
  hipLaunchKernelGGL((pack_mxfp4_kernel<TW, GU>), grid, dim3(256), 0, s,                       \
                     static_cast<const TW*>(w0), static_cast<const TW*>(w1), kdim, cols, packed, exps)
  if (w_dtype == HMOE_F32 && gate_up) HMOE_LAUNCH_PACK4(float, true);
  else if (w_dtype == HMOE_F32) HMOE_LAUNCH_PACK4(float, false);
  else if (gate_up) HMOE_LAUNCH_PACK4(uint16_t, true);
  else HMOE_LAUNCH_PACK4(uint16_t, false);
#undef HMOE_LAUNCH_PACK4
  return check_launch(what);
}

// The sizes that every packed MXFP4 operand has: whole 128-value groups of the
// reduction, rows in blocks of 32 (gate/up: 64), and the products' limits.
int check_operand(const char* what, int n_experts, int d_model, int d_ff) {
  HMOE_REQUIRE(n_experts >= 1 && n_experts <= 1024, "%s: n_experts must be in [1, 1024] (got %d)", what,
               n_experts);
  HMOE_REQUIRE_CODE(d_model >= 128 && d_model % 128 == 0 && d_model <= (1 << 20), HMOE_ERR_UNSUPPORTED,
                    "%s: d_model must be a multiple of 128 up to 2^20 (got %d)", what, d_model);
  HMOE_REQUIRE_CODE(d_ff >= 128 && d_ff % 128 == 0 && d_ff <= (1 << 20), HMOE_ERR_UNSUPPORTED,
                    "%s: d_ff must be a multiple of 128 up to 2^20 (got %d)", what, d_ff);
  return HMOE_OK;
}

}  // namespace
}  // namespace hmoe

extern "C" int hmoe_quantize_rows_mxfp4(const void* a, int a_dtype, int64_t rows, int cols, uint8_t* q,
                                        uint8_t* exps, hmoe_stream_t stream) {
  using namespace hmoe;
  HMOE_REQUIRE(rows >= 0, "quantize_rows_mxfp4: rows must be >= 0");
  HMOE_REQUIRE_CODE(cols >= kMxBlock && cols % kMxBlock == 0, HMOE_ERR_UNSUPPORTED,
                    "quantize_rows_mxfp4: cols must be a multiple of 32 (got %d)", cols);
  HMOE_REQUIRE(a_dtype == HMOE_F32 || a_dtype == HMOE_BF16,
               "quantize_rows_mxfp4: a dtype must be F32 or BF16");
  if (rows == 0) return HMOE_OK;
  HMOE_REQUIRE(a && q && exps, "quantize_rows_mxfp4: null pointer argument");
  HMOE_REQUIRE_ALIGNED("quantize_rows_mxfp4", 16, a, q);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t chunks = rows * (cols / 8);
  if (a_dtype == HMOE_BF16)
    hipLaunchKernelGGL(quantize_rows_mxfp4_kernel<uint16_t>, dim3(chunk_grid(chunks)), dim3(256), 0, s,
                       static_cast<const uint16_t*>(a), chunks, q, exps);
  else
    hipLaunchKernelGGL(quantize_rows_mxfp4_kernel<float>, dim3(chunk_grid(chunks)), dim3(256), 0, s,
                       static_cast<const float*>(a), chunks, q, exps);
  return check_launch("hmoe_quantize_rows_mxfp4");
}

extern "C" int hmoe_dequantize_rows_mxfp4(const uint8_t* q, const uint8_t* exps, int64_t rows, int cols,
                                          void* out, int out_dtype, hmoe_stream_t stream) {
  using namespace hmoe;
  HMOE_REQUIRE(rows >= 0, "dequantize_rows_mxfp4: rows must be >= 0");
  HMOE_REQUIRE_CODE(cols >= kMxBlock && cols % kMxBlock == 0, HMOE_ERR_UNSUPPORTED,
                    "dequantize_rows_mxfp4: cols must be a multiple of 32 (got %d)", cols);
  HMOE_REQUIRE(out_dtype == HMOE_F32 || out_dtype == HMOE_BF16,
               "dequantize_rows_mxfp4: out dtype must be F32 or BF16");
  if (rows == 0) return HMOE_OK;
  HMOE_REQUIRE(q && exps && out, "dequantize_rows_mxfp4: null pointer argument");
  HMOE_REQUIRE_ALIGNED("dequantize_rows_mxfp4", 16, q, out);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t chunks = rows * (cols / 8);
  const bool past = rows * cols * (out_dtype == HMOE_F32 ? 4 : 2) > kCachedBytes;
#define HMOE_LAUNCH_DEQUANT4(TO, PAST)                                                                        \
  hipLaunchKernelGGL((dequantize_rows_mxfp4_kernel<TO, PAST>), dim3(chunk_grid(chunks)), dim3(256), 0, s, q, \
                     exps, chunks, static_cast<TO*>(out))
  if (out_dtype == HMOE_F32 && past) HMOE_LAUNCH_DEQUANT4(float, true);
  else if (out_dtype == HMOE_F32) HMOE_LAUNCH_DEQUANT4(float, false);
  else if (past) HMOE_LAUNCH_DEQUANT4(uint16_t, true);
  else HMOE_LAUNCH_DEQUANT4(uint16_t, false);
#undef HMOE_LAUNCH_DEQUANT4
  return check_launch("hmoe_dequantize_rows_mxfp4");
}

extern "C" size_t hmoe_packed_mxfp4_gate_up_bytes(int n_experts, int d_model, int d_ff) {
  if (n_experts <= 0 || d_model <= 0 || d_ff <= 0) return 0;
  return static_cast<size_t>(n_experts) * d_ff * d_model;
}

extern "C" size_t hmoe_packed_mxfp4_down_bytes(int n_experts, int d_ff, int d_model) {
  if (n_experts <= 0 || d_model <= 0 || d_ff <= 0) return 0;
  return static_cast<size_t>(n_experts) * d_model * (d_ff / 2);
}

extern "C" int hmoe_pack_mxfp4_gate_up(const void* w_gate, const void* w_up, int w_dtype, int n_experts,
                                       int d_model, int d_ff, uint8_t* packed, uint8_t* exps,
                                       hmoe_stream_t stream) {
  using namespace hmoe;
  if (int rc = check_operand("pack_mxfp4_gate_up", n_experts, d_model, d_ff)) return rc;
  HMOE_REQUIRE(w_dtype == HMOE_F32 || w_dtype == HMOE_BF16,
               "pack_mxfp4_gate_up: weight dtype must be F32 or BF16");
  HMOE_REQUIRE(w_gate && w_up && packed && exps, "pack_mxfp4_gate_up: null pointer argument");
  HMOE_REQUIRE_ALIGNED("pack_mxfp4_gate_up", 16, w_gate, w_up, packed);
  HMOE_REQUIRE_ALIGNED("pack_mxfp4_gate_up", 4, exps);
  return pack_mxfp4("hmoe_pack_mxfp4_gate_up", w_gate, w_up, w_dtype, n_experts, d_model, d_ff, packed, exps,
                    static_cast<hipStream_t>(stream));
}

extern "C" int hmoe_pack_mxfp4_down(const void* w_down, int w_dtype, int n_experts, int d_ff, int d_model,
                                    uint8_t* packed, uint8_t* exps, hmoe_stream_t stream) {
  using namespace hmoe;
  if (int rc = check_operand("pack_mxfp4_down", n_experts, d_model, d_ff)) return rc;
  HMOE_REQUIRE(w_dtype == HMOE_F32 || w_dtype == HMOE_BF16, "pack_mxfp4_down: weight dtype must be F32 or BF16");
  HMOE_REQUIRE(w_down && packed && exps, "pack_mxfp4_down: null pointer argument");
  HMOE_REQUIRE_ALIGNED("pack_mxfp4_down", 16, w_down, packed);
  HMOE_REQUIRE_ALIGNED("pack_mxfp4_down", 4, exps);
  return pack_mxfp4("hmoe_pack_mxfp4_down", w_down, nullptr, w_dtype, n_experts, d_ff, d_model, packed, exps,
                    static_cast<hipStream_t>(stream));
}

extern "C" int hmoe_unpack_mxfp4(const uint8_t* packed, const uint8_t* exps, int n_experts, int rows, int cols,
                                 void* out, int out_dtype, hmoe_stream_t stream) {
  using namespace hmoe;
  HMOE_REQUIRE(n_experts >= 1 && n_experts <= 1024, "unpack_mxfp4: n_experts must be in [1, 1024] (got %d)",
               n_experts);
  HMOE_REQUIRE_CODE(rows >= 32 && rows % 32 == 0, HMOE_ERR_UNSUPPORTED,
                    "unpack_mxfp4: rows must be a multiple of 32 (got %d)", rows);
  HMOE_REQUIRE_CODE(cols >= 128 && cols % 128 == 0, HMOE_ERR_UNSUPPORTED,
                    "unpack_mxfp4: cols must be a multiple of 128 (got %d)", cols);
  HMOE_REQUIRE(out_dtype == HMOE_F32 || out_dtype == HMOE_BF16, "unpack_mxfp4: out dtype must be F32 or BF16");
  HMOE_REQUIRE(packed && exps && out, "unpack_mxfp4: null pointer argument");
  HMOE_REQUIRE_ALIGNED("unpack_mxfp4", 16, packed, out);
  const int64_t row_blocks = static_cast<int64_t>(n_experts) * (rows / 32);
  const int64_t col_blocks = ceil_div(cols / 64, kUnpackBlocks);
  // (a launch has fewer than 2^32 threads along x)
  HMOE_REQUIRE(row_blocks * 256 < (int64_t(1) << 32) && col_blocks <= 65535, "unpack_mxfp4: operand too large");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(row_blocks), static_cast<unsigned>(col_blocks));
  const bool past = row_blocks * 32 * cols * (out_dtype == HMOE_F32 ? 4 : 2) > kCachedBytes;
#define HMOE_LAUNCH_UNPACK4(TO, PAST)                                                                      \
  hipLaunchKernelGGL((unpack_mxfp4_kernel<TO, PAST>), grid, dim3(256), 0, s, packed, exps, rows, cols, \
                     static_cast<TO*>(out))
  if (out_dtype == HMOE_F32 && past) HMOE_LAUNCH_UNPACK4(float, true);
  else if (out_dtype == HMOE_F32) HMOE_LAUNCH_UNPACK4(float, false);
  else if (past) HMOE_LAUNCH_UNPACK4(uint16_t, true);
  else HMOE_LAUNCH_UNPACK4(uint16_t, false);
#undef HMOE_LAUNCH_UNPACK4
  return check_launch("hmoe_unpack_mxfp4");
}
