// Grouped products of MXFP4 rows with MXFP4 expert weights (model/moe.py:67-74 on
// 4-bit operands; the reference has no such path):
//
//   C[r, n] = sum_k A[r, k] * B_e[n, k]     for rows r of expert e's segment
//
// on v_mfma_scale_f32_32x32x64_f8f6f4, whose operands carry a power-of-two scale
// per 32 values of the reduction: products of two e2m1 values times a power of two
// are exact in float32, so what is rounded is the float32 sums and the result.  The
// gate/up product applies the SwiGLU to the float32 sums and quantises h straight
// from them (quant_mxfp4.h): h is rounded once, to four bits, and any rounding
// before that would only move values across that one's borders.
//
// The operand keeps a lane's 16 bytes of a fragment together: lane 32 h + r of
// block (p / 32, k / 64) has the 32 codes of row r from column 32 h on, so a
// fragment is one 1 KB run of memory, and its exponents [K / 128][rows][4] give
// the lanes of a fragment one run of 128 bytes per 128 columns.
#include "quant_mxfp4.h"

namespace hmoe {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kBufferWord3 = 0x00020000;

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pack_bf16x2_rne(float lo, float hi) {
  f32x2_t v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
}

// silu(g) u; the hardware's exponential and reciprocal are off by about one
// float32 step each.
__device__ __forceinline__ float swiglu_f32(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.0f + __expf(-g)) * u;
}

// One 32 x 32 x 64 product of e2m1 fragments (16 bytes a lane).  Q: the byte of
// the lanes' exponent words that holds this step's block.
template <int Q>
__device__ __forceinline__ f32x16 mfma_fp4(const u32x4& b, const u32x4& a, const f32x16& c, int eb, int ea) {
  const i32x8 b8 = {static_cast<int>(b[0]), static_cast<int>(b[1]), static_cast<int>(b[2]),
                    static_cast<int>(b[3]), 0, 0, 0, 0};
  const i32x8 a8 = {static_cast<int>(a[0]), static_cast<int>(a[1]), static_cast<int>(a[2]),
                    static_cast<int>(a[3]), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b8, a8, c, 4, 4, Q, eb, Q, ea);
}

// Segment and row tile of the m_tile-th tile of `bm` rows; false past the last.
// A wave looks at 64 experts at a time.
struct RowTile {
  int e, row0, rows;
};
__device__ __forceinline__ bool find_row_tile(const int32_t* __restrict__ offsets, int n_experts, int bm,
                                              int m_tile, RowTile& t) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int base = 0; base < n_experts; base += 64) {
    const int e = base + lane;
    const int lo = e < n_experts ? offsets[e] : 0;
    const int hi = e < n_experts ? offsets[e + 1] : 0;
    const int tiles = (hi - lo + bm - 1) / bm;
    int sum = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(sum, d);
      sum += lane >= d ? up : 0;
    }
    const int total = lane_bcast(sum, 63);
    if (m_tile < before + total) {
      // the first lane whose running count passes m_tile
      const uint64_t past = __ballot(before + sum > m_tile);
      const int src = __builtin_ctzll(past);
      const int within = m_tile - before - lane_bcast(sum - tiles, src);
      const int lo_s = lane_bcast(lo, src), hi_s = lane_bcast(hi, src);
      t.e = base + src;
      t.row0 = lo_s + within * bm;
      t.rows = hi_s - t.row0 < bm ? hi_s - t.row0 : bm;
      return true;
    }
    before += total;
  }
  return false;
}

// Epilogues.  Lane L of an accumulator holds row L % 32 of A's fragment and
// columns 8 q + 4 (L / 32) + 0..3 (q = 0..3) of B's.  Stores go through a buffer
// whose range ends at the segment's last row.
//
// h of 32 columns: gate in g, up in u; one scale block of the row.
__device__ __forceinline__ void store_h_block(const f32x16& g, const f32x16& u, __amdgpu_buffer_rsrc_t q_out,
                                              __amdgpu_buffer_rsrc_t e_out, int row, int hcol, int d_ff,
                                              int half) {
  float h[16];
  uint32_t amax = 0;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    h[k] = swiglu_f32(g[k], u[k]);
    const uint32_t b = __float_as_uint(h[k]) & 0x7fffffffu;
    amax = amax > b ? amax : b;
  }
  // lanes L and L + 32 hold the row's other values
  const auto sw = __builtin_amdgcn_permlane32_swap(amax, amax, false, false);
  const uint32_t e = mxfp4_exponent(sw[0] > sw[1] ? sw[0] : sw[1]);
  const float inv = mxfp4_inverse(e);
  uint32_t w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = h[8 * j + k];
    w[j] = mxfp4_codes8(v, inv);
  }
  // w[0] has this lane's halves of dwords 0 and 1 of the row's 16 bytes, w[1] of 2
  // and 3; lanes 0..31 take dwords 0 and 1, lanes 32..63 the others
  const auto t = __builtin_amdgcn_permlane32_swap(w[0], w[1], false, false);
  const u32x2_t d = {(t[0] & 0xffffu) | (t[1] << 16), (t[0] >> 16) | (t[1] & 0xffff0000u)};
  __builtin_amdgcn_raw_buffer_store_b64(d, q_out, (row * d_ff + hcol) / 2 + 8 * half, 0, 0);
  if (half == 0)
    __builtin_amdgcn_raw_buffer_store_b8(static_cast<uint8_t>(e), e_out, row * (d_ff / 32) + hcol / 32, 0, 0);
}

// 32 bf16 columns of a row: lanes L and L + 32 trade groups, so that each stores
// two runs of 16 bytes.
__device__ __forceinline__ void store_y_block(const f32x16& y, __amdgpu_buffer_rsrc_t out, int row, int col,
                                              int ldc, int half) {
  uint32_t d[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) d[k] = pack_bf16x2_rne(y[2 * k], y[2 * k + 1]);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const auto p01 = __builtin_amdgcn_permlane32_swap(d[w], d[2 + w], false, false);
    d[w] = p01[0];
    d[2 + w] = p01[1];
    const auto p23 = __builtin_amdgcn_permlane32_swap(d[4 + w], d[6 + w], false, false);
    d[4 + w] = p23[0];
    d[6 + w] = p23[1];
  }
  const int off = (row * ldc + col + half * 8) * 2;
  const u32x4 lo = {d[0], d[1], d[2], d[3]};
  const u32x4 hi = {d[4], d[5], d[6], d[7]};
  __builtin_amdgcn_raw_buffer_store_b128(lo, out, off, 0, 0);
  __builtin_amdgcn_raw_buffer_store_b128(hi, out, off + 32, 0, 0);
}

// A wave: 32 rows x 64 columns, operands straight from memory into registers.
// Four waves side by side.
template <bool GATE_UP, bool GATHER>
__global__ __launch_bounds__(256) void grouped_mxfp4_rows(
    const uint8_t* __restrict__ A, const uint8_t* __restrict__ a_exp, const uint8_t* __restrict__ B,
    const uint8_t* __restrict__ b_exp, const int32_t* __restrict__ offsets, int n_experts, int kdim, int ncols,
    uint8_t* __restrict__ C, uint8_t* __restrict__ c_exp, const int32_t* __restrict__ gather_src, int gather_k,
    int gather_rows) {
  const int lane = threadIdx.x & 63;
  const int frow = lane & 31, half = lane >> 5;
  RowTile t;
  if (!find_row_tile(offsets, n_experts, 32, blockIdx.y, t)) return;
  const int n0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 64;
  if (n0 >= ncols) return;
  int src = t.row0 + (frow < t.rows ? frow : t.rows - 1);  // rows past the segment repeat its last one
  if (GATHER) {
    const int slot = gather_src[src];
    src = slot >= 0 ? slot / gather_k : 0;  // a row without a source reads token 0
    src = src < gather_rows ? src : gather_rows - 1;
  }
  const int groups = kdim / 128;
  const uint8_t* a = A + static_cast<int64_t>(src) * (kdim / 2) + half * 16;
  const uint8_t* ae = a_exp + static_cast<int64_t>(src) * (kdim / 32);
  const int64_t frag = (static_cast<int64_t>(t.e) * (ncols / 32) + n0 / 32) * (kdim / 64);
  const uint8_t* b0 = B + frag * 1024 + lane * 16;
  const uint8_t* b1 = b0 + static_cast<int64_t>(kdim / 64) * 1024;
  const uint8_t* be = b_exp + (static_cast<int64_t>(t.e) * groups * ncols + n0 + frow) * 4;
  f32x16 acc0 = {}, acc1 = {};
  for (int k = 0; k < groups; ++k) {
    u32x4 fa[2], f0[2], f1[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      fa[q] = *reinterpret_cast<const u32x4*>(a + k * 64 + q * 32);
      f0[q] = *reinterpret_cast<const u32x4*>(b0 + k * 2048 + q * 1024);
      f1[q] = *reinterpret_cast<const u32x4*>(b1 + k * 2048 + q * 1024);
    }
    // byte 0 (2) of the shifted words: this lane's block of the first (second) 64
    const int ea = static_cast<int>(*reinterpret_cast<const uint32_t*>(ae + k * 4) >> (8 * half));
    const uint8_t* bk = be + static_cast<int64_t>(k) * ncols * 4;
    const int e0 = static_cast<int>(*reinterpret_cast<const uint32_t*>(bk) >> (8 * half));
    const int e1 = static_cast<int>(*reinterpret_cast<const uint32_t*>(bk + 128) >> (8 * half));
    acc0 = mfma_fp4<0>(f0[0], fa[0], acc0, e0, ea);
    acc1 = mfma_fp4<0>(f1[0], fa[0], acc1, e1, ea);
    acc0 = mfma_fp4<2>(f0[1], fa[1], acc0, e0, ea);
    acc1 = mfma_fp4<2>(f1[1], fa[1], acc1, e1, ea);
  }
  const int64_t r0 = t.row0;
  if constexpr (GATE_UP) {
    const int d_ff = ncols / 2;
    const __amdgpu_buffer_rsrc_t q_out =
        __builtin_amdgcn_make_buffer_rsrc(C + r0 * (d_ff / 2), 0, t.rows * (d_ff / 2), kBufferWord3);
    const __amdgpu_buffer_rsrc_t e_out =
        __builtin_amdgcn_make_buffer_rsrc(c_exp + r0 * (d_ff / 32), 0, t.rows * (d_ff / 32), kBufferWord3);
    store_h_block(acc0, acc1, q_out, e_out, frow, n0 / 2, d_ff, half);
  } else {
    const __amdgpu_buffer_rsrc_t out =
        __builtin_amdgcn_make_buffer_rsrc(C + r0 * ncols * 2, 0, t.rows * ncols * 2, kBufferWord3);
    store_y_block(acc0, out, frow, n0, ncols, half);
    store_y_block(acc1, out, frow, n0 + 32, ncols, half);
  }
}

// The checks that the products share.
int check_product(const char* what, int n_experts, int64_t rows_cap, int d_model, int d_ff) {
  HMOE_REQUIRE(n_experts >= 1 && n_experts <= kMaxExperts, "%s: n_experts must be in [1, %d] (got %d)", what,
               kMaxExperts, n_experts);
  HMOE_REQUIRE(rows_cap >= 0 && rows_cap < (int64_t(1) << 31), "%s: rows_cap must be in [0, 2^31)", what);
  HMOE_REQUIRE_CODE(d_model >= 128 && d_model % 128 == 0 && d_model <= (1 << 20), HMOE_ERR_UNSUPPORTED,
                    "%s: d_model must be a multiple of 128 up to 2^20 (got %d)", what, d_model);
  HMOE_REQUIRE_CODE(d_ff >= 128 && d_ff % 128 == 0 && d_ff <= (1 << 20), HMOE_ERR_UNSUPPORTED,
                    "%s: d_ff must be a multiple of 128 up to 2^20 (got %d)", what, d_ff);
  return HMOE_OK;
}

template <bool GATE_UP, bool GATHER>
int launch_product(const char* what, const uint8_t* a, const uint8_t* a_exp, const uint8_t* b,
                   const uint8_t* b_exp, const int32_t* offsets, int n_experts, int64_t rows_cap, int kdim,
                   int ncols, uint8_t* c, uint8_t* c_exp, const int32_t* gather_src, int gather_k,
                   int gather_rows, hipStream_t s) {
  // an expert's last tile may hold one row
  const int64_t full = ceil_div(rows_cap, 32) + n_experts;
  const int64_t m_tiles = full < rows_cap ? full : rows_cap;
  HMOE_REQUIRE(m_tiles <= 65535, "%s: too many row tiles", what);
  hipLaunchKernelGGL((grouped_mxfp4_rows<GATE_UP, GATHER>),
                     dim3(static_cast<unsigned>(ceil_div(ncols, 256)), static_cast<unsigned>(m_tiles)), dim3(256),
                     0, s, a, a_exp, b, b_exp, offsets, n_experts, kdim, ncols, c, c_exp, gather_src, gather_k,
                     gather_rows);
  return check_launch(what);
}

}  // namespace
}  // namespace hmoe

extern "C" int hmoe_grouped_gate_up_mxfp4(const uint8_t* xs_q, const uint8_t* xs_exp, const int32_t* offsets,
                                          int n_experts, int64_t rows_cap, int d_model, int d_ff,
                                          const uint8_t* w_packed, const uint8_t* w_exp, uint8_t* h_q,
                                          uint8_t* h_exp, hmoe_stream_t stream) {
  using namespace hmoe;
  const char* what = "grouped_gate_up_mxfp4";
  if (int rc = check_product(what, n_experts, rows_cap, d_model, d_ff)) return rc;
  if (rows_cap == 0) return HMOE_OK;
  HMOE_REQUIRE(xs_q && xs_exp && offsets && w_packed && w_exp && h_q && h_exp, "%s: null pointer argument", what);
  HMOE_REQUIRE_ALIGNED(what, xs_q, xs_exp, w_packed, w_exp, h_q);
  return launch_product<true, false>(what, xs_q, xs_exp, w_packed, w_exp, offsets, n_experts, rows_cap, d_model,
                                     2 * d_ff, h_q, h_exp, nullptr, 1, 1, static_cast<hipStream_t>(stream));
}

extern "C" int hmoe_grouped_gate_up_mxfp4_gather(const uint8_t* x_q, const uint8_t* x_exp, int64_t tokens,
                                                 int top_k, const int32_t* perm_src, const int32_t* offsets,
                                                 int n_experts, int64_t rows_cap, int d_model, int d_ff,
                                                 const uint8_t* w_packed, const uint8_t* w_exp, uint8_t* h_q,
                                                 uint8_t* h_exp, hmoe_stream_t stream) {
  using namespace hmoe;
  const char* what = "grouped_gate_up_mxfp4_gather";
  if (int rc = check_product(what, n_experts, rows_cap, d_model, d_ff)) return rc;
  HMOE_REQUIRE(tokens >= 0 && top_k >= 1 && (tokens >= 1 || rows_cap == 0),
               "%s: need tokens >= 0, top_k >= 1 (tokens >= 1 with rows)", what);
  HMOE_REQUIRE(tokens < (int64_t(1) << 31) && tokens * (d_model / 2) < (int64_t(1) << 31),
               "%s: x_q must be smaller than 2 GiB", what);
  if (rows_cap == 0) return HMOE_OK;
  HMOE_REQUIRE(x_q && x_exp && perm_src && offsets && w_packed && w_exp && h_q && h_exp,
               "%s: null pointer argument", what);
  HMOE_REQUIRE_ALIGNED(what, x_q, x_exp, w_packed, w_exp, h_q);
  return launch_product<true, true>(what, x_q, x_exp, w_packed, w_exp, offsets, n_experts, rows_cap, d_model,
                                    2 * d_ff, h_q, h_exp, perm_src, top_k, static_cast<int>(tokens),
                                    static_cast<hipStream_t>(stream));
}

extern "C" int hmoe_grouped_down_mxfp4(const uint8_t* h_q, const uint8_t* h_exp, const int32_t* offsets,
                                       int n_experts, int64_t rows_cap, int d_ff, int d_model,
                                       const uint8_t* w_packed, const uint8_t* w_exp, void* ys,
                                       hmoe_stream_t stream) {
  using namespace hmoe;
  const char* what = "grouped_down_mxfp4";
  if (int rc = check_product(what, n_experts, rows_cap, d_model, d_ff)) return rc;
  if (rows_cap == 0) return HMOE_OK;
  HMOE_REQUIRE(h_q && h_exp && offsets && w_packed && w_exp && ys, "%s: null pointer argument", what);
  HMOE_REQUIRE_ALIGNED(what, h_q, h_exp, w_packed, w_exp, ys);
  return launch_product<false, false>(what, h_q, h_exp, w_packed, w_exp, offsets, n_experts, rows_cap, d_ff,
                                      d_model, static_cast<uint8_t*>(ys), nullptr, nullptr, 1, 1,
                                      static_cast<hipStream_t>(stream));
}
