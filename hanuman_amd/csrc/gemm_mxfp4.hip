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
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "quant_mxfp4.h"

namespace hmoe {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int64_t kMaxRows = int64_t(1) << 30;
constexpr int kBufferWord3 = 0x00020000;
constexpr int kNonTemporal = 2;  // cache policy of a buffer access

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

// Epilogues.  Lane L of an accumulator holds row L % 32 of A's fragment and columns 8 q
// + 4 (L / 32) + 0..3 (q = 0..3) of B's.  Stores go through a buffer whose range ends
// at the segment's last row.
//
// h of 32 columns (gate in g, up in u), one scale block of the row: its exponent, and in
// w[0] this lane's halves of dwords 0 and 1 of the row's 16 bytes of codes, in w[1] of
// dwords 2 and 3.
__device__ __forceinline__ uint32_t quantise_h(const f32x16& g, const f32x16& u, uint32_t (&w)[2]) {
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
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = h[8 * j + k];
    w[j] = mxfp4_codes8(v, inv);
  }
  return e;
}
// The halves of lanes L (lo) and L + 32 (hi) put together.
__device__ __forceinline__ u32x2_t join_codes(uint32_t lo, uint32_t hi) {
  return u32x2_t{(lo & 0xffffu) | (hi << 16), (lo >> 16) | (hi & 0xffff0000u)};
}

// One block: lanes 0..31 store dwords 0 and 1 of their row, lanes 32..63 the others.
__device__ __forceinline__ void store_h_block(const f32x16& g, const f32x16& u, __amdgpu_buffer_rsrc_t q_out,
                                              __amdgpu_buffer_rsrc_t e_out, int row, int hcol, int d_ff,
                                              int half) {
  uint32_t w[2];
  const uint32_t e = quantise_h(g, u, w);
  const auto t = __builtin_amdgcn_permlane32_swap(w[0], w[1], false, false);
  __builtin_amdgcn_raw_buffer_store_b64(join_codes(t[0], t[1]), q_out, (row * d_ff + hcol) / 2 + 8 * half, 0, 0);
  if (half == 0)
    __builtin_amdgcn_raw_buffer_store_b8(static_cast<uint8_t>(e), e_out, row * (d_ff / 32) + hcol / 32, 0, 0);
}

// Two blocks side by side: lanes 0..31 store the first's 16 bytes of their row and both
// exponents, lanes 32..63 the second's.
__device__ __forceinline__ void store_h_blocks(const f32x16 (&acc)[4], __amdgpu_buffer_rsrc_t q_out,
                                               __amdgpu_buffer_rsrc_t e_out, int row, int hcol, int d_ff,
                                               int half) {
  uint32_t w0[2], w1[2];
  const uint32_t e0 = quantise_h(acc[0], acc[1], w0);
  const uint32_t e1 = quantise_h(acc[2], acc[3], w1);
  // (lanes 0..31 give their halves of block 1 for the others' of block 0)
  const auto a = __builtin_amdgcn_permlane32_swap(w0[0], w1[0], false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(w0[1], w1[1], false, false);
  const u32x2_t lo = join_codes(a[0], a[1]), hi = join_codes(b[0], b[1]);
  const u32x4 codes = {lo[0], lo[1], hi[0], hi[1]};
  __builtin_amdgcn_raw_buffer_store_b128(codes, q_out, (row * d_ff + hcol) / 2 + 16 * half, 0, 0);
  if (half == 0)
    __builtin_amdgcn_raw_buffer_store_b16(static_cast<uint16_t>(e0 | (e1 << 8)), e_out,
                                          row * (d_ff / 32) + hcol / 32, 0, 0);
}

// 32 bf16 columns of a row: lanes L and L + 32 trade groups, after which lane L < 32
// holds columns 0..7 and 16..23 of its row, lane L + 32 columns 8..15 and 24..31.
__device__ __forceinline__ void pack_y_block(const f32x16& y, u32x4& lo, u32x4& hi) {
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
  lo = u32x4{d[0], d[1], d[2], d[3]};
  hi = u32x4{d[4], d[5], d[6], d[7]};
}
__device__ __forceinline__ void store_y_block(const f32x16& y, __amdgpu_buffer_rsrc_t out, int row, int col,
                                              int ldc, int half) {
  u32x4 lo, hi;
  pack_y_block(y, lo, hi);
  const int off = (row * ldc + col + half * 8) * 2;
  __builtin_amdgcn_raw_buffer_store_b128(lo, out, off, 0, 0);
  __builtin_amdgcn_raw_buffer_store_b128(hi, out, off + 32, 0, 0);
}

// Two blocks side by side (64 columns, 32 rows), through 4 KB of LDS that only this
// wave uses, so that a store instruction writes whole 128-byte lines: chunk c of row r
// sits at c ^ (r & 7).  ys is far larger than the caches where tiles are taken, and kept
// out of them: at 131072 x 2048 outputs of 1024 values the product takes 287 us with
// 32-byte stores from the accumulators, 245 us with whole lines, 187 us with whole lines
// that are not cached.
__device__ __forceinline__ void store_y_blocks(const f32x16& y0, const f32x16& y1, uint8_t* lds,
                                               __amdgpu_buffer_rsrc_t out, int row0, int col, int ldc, int lane) {
  const int r = lane & 31, half = lane >> 5;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    u32x4 lo, hi;
    pack_y_block(j == 0 ? y0 : y1, lo, hi);
    uint8_t* p = lds + r * 128;
    *reinterpret_cast<u32x4*>(p + (((4 * j + half) ^ (r & 7)) * 16)) = lo;
    *reinterpret_cast<u32x4*>(p + (((4 * j + 2 + half) ^ (r & 7)) * 16)) = hi;
  }
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const int rr = 8 * m + (lane >> 3);
    const u32x4 v = *reinterpret_cast<const u32x4*>(lds + rr * 128 + (((lane & 7) ^ (rr & 7)) * 16));
    __builtin_amdgcn_raw_buffer_store_b128(v, out, ((row0 + rr) * ldc + col + (lane & 7) * 8) * 2, 0, kNonTemporal);
  }
}

// ---- few rows ---------------------------------------------------------------------
// 32 rows x 64 columns a wave, operands straight from memory into registers: with few
// rows an expert every weight is used once or twice, and a fragment is one run of 1 KB.
// Four groups of 128 values are loaded together, so that a wave has 20 KB on the way.
// A workgroup is four waves: side by side (SPLIT 1), or on a quarter of the reduction
// each, joined in LDS in their order (SPLIT 4).  The split shortens the one chain of
// loads that a call of few tiles consists of.
template <bool GATE_UP, bool GATHER, int SPLIT>
__global__ __launch_bounds__(256) void grouped_mxfp4_rows(
    const uint8_t* __restrict__ A, const uint8_t* __restrict__ a_exp, const uint8_t* __restrict__ B,
    const uint8_t* __restrict__ b_exp, const int32_t* __restrict__ offsets, int n_experts, int kdim, int ncols,
    uint8_t* __restrict__ C, uint8_t* __restrict__ c_exp, const int32_t* __restrict__ gather_src, int gather_k,
    int gather_rows) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int frow = lane & 31, half = lane >> 5;
  RowTile t;
  if (!find_row_tile(offsets, n_experts, 32, blockIdx.y, t)) return;
  const int n0 = SPLIT == 1 ? (blockIdx.x * 4 + wave) * 64 : blockIdx.x * 64;
  if (n0 >= ncols) return;  // (SPLIT 1 only: no barrier follows there)
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
  struct Group {
    u32x4 fa[2], f0[2], f1[2];
    uint32_t ea, e0, e1;
  };
  auto load = [&](Group& p, int k) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      p.fa[q] = *reinterpret_cast<const u32x4*>(a + k * 64 + q * 32);
      p.f0[q] = *reinterpret_cast<const u32x4*>(b0 + static_cast<int64_t>(k) * 2048 + q * 1024);
      p.f1[q] = *reinterpret_cast<const u32x4*>(b1 + static_cast<int64_t>(k) * 2048 + q * 1024);
    }
    const uint8_t* bk = be + static_cast<int64_t>(k) * ncols * 4;
    p.ea = *reinterpret_cast<const uint32_t*>(ae + k * 4);
    p.e0 = *reinterpret_cast<const uint32_t*>(bk);
    p.e1 = *reinterpret_cast<const uint32_t*>(bk + 128);
  };
  auto use = [&](const Group& p) __attribute__((always_inline)) {
    // byte 0 (2) of the shifted words: this lane's block of the first (second) 64
    const int ea = static_cast<int>(p.ea >> (8 * half));
    const int e0 = static_cast<int>(p.e0 >> (8 * half));
    const int e1 = static_cast<int>(p.e1 >> (8 * half));
    acc0 = mfma_fp4<0>(p.f0[0], p.fa[0], acc0, e0, ea);
    acc1 = mfma_fp4<0>(p.f1[0], p.fa[0], acc1, e1, ea);
    acc0 = mfma_fp4<2>(p.f0[1], p.fa[1], acc0, e0, ea);
    acc1 = mfma_fp4<2>(p.f1[1], p.fa[1], acc1, e1, ea);
  };
  int k = SPLIT == 1 ? 0 : groups * wave / SPLIT;
  const int end = SPLIT == 1 ? groups : groups * (wave + 1) / SPLIT;
  for (; k + 4 <= end; k += 4) {
    Group p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) load(p[j], k + j);
#pragma unroll
    for (int j = 0; j < 4; ++j) use(p[j]);
  }
  for (; k < end; ++k) {
    Group p;
    load(p, k);
    use(p);
  }
  if constexpr (SPLIT > 1) {
    // wave 0 adds the others' sums, in their order
    __shared__ f32x4 part[SPLIT - 1][8][64];
    if (wave > 0) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        part[wave - 1][r][lane] = f32x4{acc0[4 * r], acc0[4 * r + 1], acc0[4 * r + 2], acc0[4 * r + 3]};
        part[wave - 1][4 + r][lane] = f32x4{acc1[4 * r], acc1[4 * r + 1], acc1[4 * r + 2], acc1[4 * r + 3]};
      }
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 0; w < SPLIT - 1; ++w)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 p0 = part[w][r][lane], p1 = part[w][4 + r][lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc0[4 * r + i] += p0[i];
          acc1[4 * r + i] += p1[i];
        }
      }
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

// ---- tiles for experts with many rows ------------------------------------------
// Two workgroups of four waves share a CU, each looping over BM x 256 tiles: while one
// is in its epilogue (the SwiGLU's exponentials and reciprocals alone take a quarter of
// the products' time), switches tiles or waits at its barrier, the other's products run.
// A K step is 128 values = 64 bytes of every row; the operands go from global memory
// into a ring of three LDS stages (buffer_load ... lds), two steps ahead and on into
// the next tile, one barrier a step.  A's part of a stage has 64-byte rows whose 16-byte
// chunk c sits at c ^ swz64(r), so that 16 lanes of a fragment read cover all banks;
// B's is the operand's own blocks of 1 KB, read lane by lane, and its exponents are a
// run of 1 KB, put down in the order in which a lane reads four words.  A's exponents, 16 bytes of every row, come for up to four steps at once
// into one of two regions (three with 64 rows, where a tile may be a single step).  The
// last column tile may be 128 columns wide: the waves of the other half load and compute
// the first half's again and store nothing.
//
// What bounds the large products is power: with these operands the matrix cores alone,
// fed from registers, run at 1.65 GHz and 6.5 PFLOP/s.  Gate/up of 131072 rows, D 2048, F
// 1024 (1.1 TFLOP) takes 333 us, 300 of them in the loop at 1.6 to 1.8 GHz, 1580 cycles for
// two workgroups' steps (1024 of MFMA).  One workgroup of eight waves on 256 x 256 tiles (a
// third less from L2) took 336 us at 1.8 GHz and 1750 cycles, four waves of 128 x 128
// (a third less from LDS too) 400 us, the 16 x 16 x 128 MFMA 1900 cycles at 1.95 GHz, all
// about 300 us in the loop.
constexpr int kTileThreads = 256;
constexpr int kStages = 3;
constexpr int kNumXcd = 8;
constexpr int kTileN = 256;
constexpr int kTileGroup = 8;

template <int BM>
struct TileCfg {
  static constexpr int kA = BM * 64, kB = kTileN * 64, kExB = kTileN * 4;
  static constexpr int kStage = kA + kB + kExB;
  static constexpr int kExA = BM * 16;
  static constexpr int kRegions = BM == 64 ? 3 : 2;
  static constexpr int kLds = kStages * kStage + kRegions * kExA;
  static constexpr int kNA = BM / 64, kNB = kTileN / 64;  // DMA instructions a wave and step
  static constexpr int kFR = BM / 64;                      // row fragments a wave
  static_assert(2 * kLds <= 160 * 1024, "two workgroups a CU");
};

typedef __attribute__((address_space(3))) void* lds_ptr_t;

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint8_t* dst, uint32_t voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)dst, 16, voff, soff, 0, 0);
}
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t r, uint8_t* dst, uint32_t voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)dst, 4, voff, soff, 0, 0);
}

// A use that later code is not moved before.  (A function of its own, like dma16:
// where the operand's type depends on a template the host pass drops the kernel.)
__device__ __forceinline__ void use_here(const f32x16& v) { asm volatile("" ::"v"(v)); }

__device__ __forceinline__ int swz64(int r) { return (r >> 2) & 3; }

// s_waitcnt vmcnt(N) lgkmcnt(0)
template <int N>
__device__ __forceinline__ void wait_vm_lgkm0() {
  static_assert(N >= 0 && N < 64, "vmcnt is a 6-bit count");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0070);
}

// Row tiles of all experts.
__device__ __forceinline__ int count_row_tiles(const int32_t* __restrict__ offsets, int n_experts, int bm) {
  const int lane = threadIdx.x & 63;
  int sum = 0;
  for (int e = lane; e < n_experts; e += 64) sum += (offsets[e + 1] - offsets[e] + bm - 1) / bm;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
  return __builtin_amdgcn_readfirstlane(sum);
}

// Where a workgroup is in the experts' tiles.  An expert's tiles are taken in groups of
// kTileGroup row tiles, each swept column by column (row tile fastest), so that an XCD's
// workgroups share few blocks of A and B.
template <int BM>
struct TileCursor {
  int e, before, tiles;  // expert, row tiles before its first, its row tiles
  int seg0, seg1;        // its rows
  int row0, rows, n0;    // the tile

  __device__ __forceinline__ void expert(const int32_t* __restrict__ offsets, int n) {
    e = n;
    seg0 = __builtin_amdgcn_readfirstlane(offsets[n]);
    seg1 = __builtin_amdgcn_readfirstlane(offsets[n + 1]);
    tiles = (seg1 - seg0 + BM - 1) / BM;
  }
  // The expert of row tile m, 64 experts at a time (m is below their row tiles).
  __device__ __forceinline__ void find(const int32_t* __restrict__ offsets, int n_experts, int m) {
    const int lane = threadIdx.x & 63;
    before = 0;
    for (int base = 0;; base += 64) {
      const int ee = base + lane;
      const int mine = ee < n_experts ? (offsets[ee + 1] - offsets[ee] + BM - 1) / BM : 0;
      int sum = mine;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int up = __shfl_up(sum, d);
        sum += lane >= d ? up : 0;
      }
      const int total = lane_bcast(sum, 63);
      if (m < before + total || base + 64 >= n_experts) {
        const uint64_t past = __ballot(before + sum > m);
        const int src = past != 0 ? __builtin_ctzll(past) : 63;
        before += lane_bcast(sum - mine, src);
        expert(offsets, base + src);
        return;
      }
      before += total;
    }
  }
  // On to tile t (t grows from call to call).
  __device__ __forceinline__ void move(const int32_t* __restrict__ offsets, int t, int n_tiles_n) {
    const int m_any = t / n_tiles_n;
    while (m_any >= before + tiles) {
      before += tiles;
      expert(offsets, e + 1);
    }
    const int u = t - before * n_tiles_n;
    const int g = u / (kTileGroup * n_tiles_n);
    const int left = tiles - g * kTileGroup;
    const int gm = left < kTileGroup ? left : kTileGroup;
    const int v = u - g * kTileGroup * n_tiles_n;
    const int n_tile = v / gm;
    row0 = seg0 + (g * kTileGroup + (v - n_tile * gm)) * BM;
    rows = seg1 - row0 < BM ? seg1 - row0 : BM;
    n0 = n_tile * kTileN;
  }
};

// Steps of the group that starts with `left` steps to go: four, but no group of one
// after another (the steps in the ring then span two groups at most).
__device__ __forceinline__ int group_steps(int left) { return left == 5 ? 3 : left < 4 ? left : 4; }

template <int BM, bool GATE_UP, bool GATHER>
__global__ __launch_bounds__(kTileThreads, 2) void grouped_mxfp4_tiles(
    const uint8_t* __restrict__ A, const uint8_t* __restrict__ a_exp, const uint8_t* __restrict__ B,
    const uint8_t* __restrict__ b_exp, const int32_t* __restrict__ offsets, int n_experts, int kdim, int ncols,
    uint8_t* __restrict__ C, uint8_t* __restrict__ c_exp, const int32_t* __restrict__ gather_src, int gather_k,
    int gather_rows) {
  typedef TileCfg<BM> Cfg;
  constexpr int kNA = Cfg::kNA, kNB = Cfg::kNB, kFR = Cfg::kFR;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n_tiles_n = (ncols + kTileN - 1) / kTileN;
  const int total = count_row_tiles(offsets, n_experts, BM) * n_tiles_n;
  // the tiles are split evenly over the XCDs (workgroup i runs on XCD i % 8)
  const int xcd = blockIdx.x % kNumXcd;
  const int per_xcd = gridDim.x / kNumXcd;
  const int lo = static_cast<int>((static_cast<int64_t>(total) * xcd) / kNumXcd);
  const int hi = static_cast<int>((static_cast<int64_t>(total) * (xcd + 1)) / kNumXcd);
  const int first = lo + static_cast<int>(blockIdx.x) / kNumXcd;
  if (first >= hi) return;  // uniform per workgroup
  const int ks = kdim / 128;
  const int row_bytes = kdim / 2, ex_bytes = kdim / 32;
  const int iters = (hi - first + per_xcd - 1) / per_xcd * ks;

  // ---- load side -----------------------------------------------------------------
  // A: instruction j of wave w fills rows 16 (w kNA + j) + lane / 4, chunk (lane & 3)
  // ^ swz64(row).  B: blocks of 1 KB, block b = 2 (column / 32) + (64 values of the
  // step), instruction j of wave w block w kNB + j; its exponents 256 bytes a wave.
  static_assert(kNB == 4, "two blocks of columns a wave");
  TileCursor<BM> ld;
  ld.find(offsets, n_experts, first / n_tiles_n);
  TileCursor<BM> cur = ld;
  const int a_row = 16 * wave * kNA + (lane >> 2);
  const int a_byte = ((lane & 3) ^ ((lane >> 4) & 3)) * 16;
  __amdgpu_buffer_rsrc_t a_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(A), 0,
                                                                    GATHER ? gather_rows * row_bytes : 0, kBufferWord3);
  __amdgpu_buffer_rsrc_t ae_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a_exp), 0,
                                                                     GATHER ? gather_rows * ex_bytes : 0, kBufferWord3);
  __amdgpu_buffer_rsrc_t b_rsrc = a_rsrc, be_rsrc = a_rsrc;
  uint32_t a_voff[kNA], ae_voff = 0;
  const int b_col = (kdim / 64) * 1024;  // bytes of 32 columns
  // (words of a half's columns c, c + 32, c + 64, c + 96 together, as a lane reads them)
  const int ex_word = (wave & 1) * 64 + lane;
  const uint32_t be_voff = static_cast<uint32_t>(((ex_word & 3) * 32 + (ex_word >> 2)) * 4);
  int b_wave = 0, be_wave = 0;       // where this wave's part of B's tile begins
  const bool ex_a = wave < BM / 64;  // the waves that bring A's exponents
  int ld_kb = 0, ld_left = 0, ld_g = 0, ld_t = first, ld_region = Cfg::kRegions - 1, ld_stage = 0;
  int32_t pf_src[kNA], pf_ex = 0;  // GATHER: sources of this lane's rows
  auto fetch_src = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kNA; ++j) {
      const int r = a_row + 16 * j;
      pf_src[j] = gather_src[ld.row0 + (r < ld.rows ? r : ld.rows - 1)];
    }
    const int r = 64 * wave + lane;
    if (ex_a) pf_ex = gather_src[ld.row0 + (r < ld.rows ? r : ld.rows - 1)];
  };
  auto token = [&](int32_t slot) __attribute__((always_inline)) {
    const int tk = slot >= 0 ? slot / gather_k : 0;  // a row without a source reads token 0
    return static_cast<uint32_t>(tk < gather_rows ? tk : gather_rows - 1);
  };
  auto set_load_tile = [&]() __attribute__((always_inline)) {
    ld.move(offsets, ld_t, n_tiles_n);
    if (GATHER) fetch_src();
    const int64_t block = static_cast<int64_t>(ld.e) * (ncols / 32) + ld.n0 / 32;
    const int width = ncols - ld.n0 < kTileN ? ncols - ld.n0 : kTileN;
    const int part = 64 * wave < width ? wave : wave - 2;  // (a tile of 128 columns: waves 0 and 1 again)
    b_wave = part * 2 * b_col;
    be_wave = (part >> 1) * 512;
    b_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(B + block * b_col), 0, width * row_bytes,
                                               kBufferWord3);
    be_rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(b_exp + (static_cast<int64_t>(ld.e) * ks * ncols + ld.n0) * 4), 0,
        ((ks - 1) * ncols + width) * 4, kBufferWord3);
    if (GATHER) {
#pragma unroll
      for (int j = 0; j < kNA; ++j) a_voff[j] = token(pf_src[j]) * static_cast<uint32_t>(row_bytes) + a_byte;
      ae_voff = token(pf_ex) * static_cast<uint32_t>(ex_bytes);
    } else {
      // rows past the segment repeat its last one; their results are not stored
      a_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(A + static_cast<int64_t>(ld.row0) * row_bytes),
                                                 0, ld.rows * row_bytes, kBufferWord3);
      ae_rsrc = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint8_t*>(a_exp + static_cast<int64_t>(ld.row0) * ex_bytes), 0, ld.rows * ex_bytes, kBufferWord3);
#pragma unroll
      for (int j = 0; j < kNA; ++j) {
        const int r = a_row + 16 * j;
        a_voff[j] = static_cast<uint32_t>((r < ld.rows ? r : ld.rows - 1) * row_bytes + a_byte);
      }
      const int r = 64 * wave + lane;
      ae_voff = static_cast<uint32_t>((r < ld.rows ? r : ld.rows - 1) * ex_bytes);
    }
    ld_kb = 0;
  };
  // One step into the ring.  (Every step loaded: the last one again, into a stage that
  // nothing reads, so that a step always issues as many.)
  auto issue = [&]() __attribute__((always_inline)) {
    if (ld_g < iters && ld_left == 0) {
      if (ld_kb == ks) {
        ld_t += per_xcd;
        set_load_tile();
      }
      ld_left = group_steps(ks - ld_kb);
      ld_region = ld_region + 1 == Cfg::kRegions ? 0 : ld_region + 1;
      // (what a short group reads past a row's end is not used; past the buffer it is
      // not read)
      if (ex_a)
        dma16(ae_rsrc, smem + kStages * Cfg::kStage + ld_region * Cfg::kExA + wave * 1024,
              ae_voff + static_cast<uint32_t>(ld_kb * 4), 0);
    }
    const int kb = ld_g < iters ? ld_kb : ld_kb - 1;
    uint8_t* st = smem + ld_stage * Cfg::kStage;
#pragma unroll
    for (int j = 0; j < kNA; ++j) dma16(a_rsrc, st + (wave * kNA + j) * 1024, a_voff[j], kb * 64);
#pragma unroll
    for (int j = 0; j < kNB; ++j)
      dma16(b_rsrc, st + Cfg::kA + (wave * kNB + j) * 1024, static_cast<uint32_t>(lane * 16),
            b_wave + (j >> 1) * b_col + kb * 2048 + (j & 1) * 1024);
    dma4(be_rsrc, st + Cfg::kA + Cfg::kB + wave * 256, be_voff, be_wave + kb * ncols * 4);
    if (ld_g < iters) {
      ++ld_g;
      ++ld_kb;
      --ld_left;
    }
    ld_stage = ld_stage + 1 == kStages ? 0 : ld_stage + 1;
  };

  // ---- compute side ----------------------------------------------------------------
  // Wave w: rows (BM / 2) (w & 1) .. and columns 128 (w >> 1) .. of the tile.
  const int wm = wave & 1, wn = wave >> 1;
  const int frow = lane & 31, half = lane >> 5;
  const int fsw = swz64(frow);
  const int a_off = (wm * (BM / 2) + frow) * 64;
  const int b_off = Cfg::kA + wn * 8192 + lane * 16;
  const int be_off = Cfg::kA + Cfg::kB + wn * 512 + frow * 16;
  const int ae_off = kStages * Cfg::kStage + (wm * (BM / 2) + frow) * 16;
  f32x16 acc[kFR][4];
  int stage = 0, region = Cfg::kRegions - 1, left = 0, in_group = 0;
  auto step = [&]() __attribute__((always_inline)) {
    const uint8_t* st = smem + stage * Cfg::kStage;
    u32x4 fa[2][kFR], fb[2][4];
    int exa[kFR], exb[4];
    const u32x4 exw = *reinterpret_cast<const u32x4*>(st + be_off);
#pragma unroll
    for (int j = 0; j < 4; ++j) exb[j] = static_cast<int>(exw[j] >> (8 * half));
#pragma unroll
    for (int i = 0; i < kFR; ++i)
      exa[i] = static_cast<int>(*reinterpret_cast<const uint32_t*>(smem + ae_off + region * Cfg::kExA + i * 512 +
                                                                   in_group * 4) >>
                                (8 * half));
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int j = 0; j < 4; ++j) fb[q][j] = *reinterpret_cast<const u32x4*>(st + b_off + j * 2048 + q * 1024);
#pragma unroll
      for (int i = 0; i < kFR; ++i)
        fa[q][i] = *reinterpret_cast<const u32x4*>(st + a_off + i * 2048 + (((2 * q + half) ^ fsw) * 16));
    }
#pragma unroll
    for (int i = 0; i < kFR; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mfma_fp4<0>(fb[0][j], fa[0][i], acc[i][j], exb[j], exa[i]);
#pragma unroll
    for (int i = 0; i < kFR; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mfma_fp4<2>(fb[1][j], fa[1][i], acc[i][j], exb[j], exa[i]);
    // used here, before the barrier, so that the products are not moved past it
#pragma unroll
    for (int i = 0; i < kFR; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) use_here(acc[i][j]);
  };

  ld.move(offsets, first, n_tiles_n);
  set_load_tile();
  issue();
  issue();
  int g = 0;
  for (int t = first; t < hi; t += per_xcd) {
#pragma unroll
    for (int i = 0; i < kFR; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    for (int kb = 0; kb < ks; ++kb, ++g) {
      // this wave's loads of step g have landed (step g + 1's may fly); after the
      // barrier every wave's have, and every wave is done with step g - 1, whose stage
      // the next loads take
      wait_vm_lgkm0<kNA + kNB + 1>();
      __builtin_amdgcn_s_barrier();
      issue();
      if (left == 0) {
        left = group_steps(ks - kb);
        region = region + 1 == Cfg::kRegions ? 0 : region + 1;
        in_group = 0;
      }
      step();
      --left;
      ++in_group;
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    cur.move(offsets, t, n_tiles_n);
    const int64_t r0 = cur.row0;
    const int row = wm * (BM / 2) + frow;
    const bool mine = cur.n0 + wn * 128 < ncols;  // uniform per wave
    if constexpr (GATE_UP) {
      const int d_ff = ncols / 2;
      const __amdgpu_buffer_rsrc_t q_out =
          __builtin_amdgcn_make_buffer_rsrc(C + r0 * (d_ff / 2), 0, cur.rows * (d_ff / 2), kBufferWord3);
      const __amdgpu_buffer_rsrc_t e_out =
          __builtin_amdgcn_make_buffer_rsrc(c_exp + r0 * (d_ff / 32), 0, cur.rows * (d_ff / 32), kBufferWord3);
#pragma unroll
      for (int i = 0; i < kFR; ++i)
        if (mine) store_h_blocks(acc[i], q_out, e_out, row + 32 * i, cur.n0 / 2 + wn * 64, d_ff, half);
    } else {
      const __amdgpu_buffer_rsrc_t out =
          __builtin_amdgcn_make_buffer_rsrc(C + r0 * ncols * 2, 0, cur.rows * ncols * 2, kBufferWord3);
      // through the stage of the last step, which every wave has read once all are here
      // and which the next step's loads take after their barrier
      uint8_t* const lds = smem + (stage == 0 ? kStages - 1 : stage - 1) * Cfg::kStage + wave * 4096;
      __builtin_amdgcn_s_barrier();
#pragma unroll
      for (int i = 0; i < kFR; ++i)
#pragma unroll
        for (int j = 0; j < 4; j += 2)
          if (mine)
            store_y_blocks(acc[i][j], acc[i][j + 1], lds, out, wm * (BM / 2) + 32 * i, cur.n0 + wn * 128 + 32 * j, ncols,
                         lane);
    }
  }
  // nothing may still be writing into LDS when the workgroup ends
  __builtin_amdgcn_s_waitcnt(0);
}

// Workgroups of a persistent launch: one a CU, a multiple of the XCDs.
int persistent_grid(const char* what, hipStream_t s, int* grid, int* dev_out) {
  int dev = 0;
  if (hipStreamGetDevice(s, &dev) != hipSuccess && hipGetDevice(&dev) != hipSuccess) {
    set_error("%s: cannot query the stream's device", what);
    return HMOE_ERR_HIP;
  }
  static std::atomic<int> cached[64];
  int cus = dev >= 0 && dev < 64 ? cached[dev].load(std::memory_order_relaxed) : 0;
  if (cus == 0) {
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) {
      set_error("%s: cannot query the CU count of device %d", what, dev);
      return HMOE_ERR_HIP;
    }
    if (dev >= 0 && dev < 64) cached[dev].store(cus, std::memory_order_relaxed);
  }
  const int g = cus / kNumXcd * kNumXcd;
  *grid = g > 0 ? g : kNumXcd;
  *dev_out = dev;
  return HMOE_OK;
}

// Allows a kernel its dynamic LDS, once per device.
template <typename Kernel>
int allow_lds(const char* what, Kernel kernel, int bytes, int dev, std::atomic<uint64_t>* done) {
  const uint64_t bit = dev >= 0 && dev < 64 ? uint64_t(1) << dev : 0;
  if (bit != 0 && (done->load(std::memory_order_acquire) & bit) != 0) return HMOE_OK;
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
      hipSuccess) {
    set_error("%s: cannot allow %d bytes of dynamic LDS on device %d", what, bytes, dev);
    return HMOE_ERR_HIP;
  }
  done->fetch_or(bit, std::memory_order_release);
  return HMOE_OK;
}

// Tiles of 32 rows at most: an expert's last one may hold a single row.
int64_t max_row_tiles(int64_t rows, int n_experts) {
  const int64_t full = ceil_div(rows, 32) + n_experts;
  return full < rows ? full : rows;
}

// The checks that the products share.
int check_product(const char* what, int n_experts, int64_t rows_cap, int d_model, int d_ff) {
  HMOE_REQUIRE(n_experts >= 1 && n_experts <= kMaxExperts, "%s: n_experts must be in [1, %d] (got %d)", what,
               kMaxExperts, n_experts);
  // (2^30: a tile's rows and the tiles that a workgroup steps over are added in 32 bits)
  HMOE_REQUIRE(rows_cap >= 0 && rows_cap <= kMaxRows, "%s: rows_cap must be in [0, 2^30]", what);
  HMOE_REQUIRE_CODE(d_model >= 128 && d_model % 128 == 0 && d_model <= (1 << 20), HMOE_ERR_UNSUPPORTED,
                    "%s: d_model must be a multiple of 128 up to 2^20 (got %d)", what, d_model);
  HMOE_REQUIRE_CODE(d_ff >= 128 && d_ff % 128 == 0 && d_ff <= (1 << 20), HMOE_ERR_UNSUPPORTED,
                    "%s: d_ff must be a multiple of 128 up to 2^20 (got %d)", what, d_ff);
  return HMOE_OK;
}

// Which kernel a product takes: the one with the least estimated time, from three
// measured rates (MI355X, us, `steps` = K / 128):
//   rows split four ways: 3.5, and 0.55 ns for every 32 rows x 64 columns x 128 values;
//   64-row tiles:  4.2 + 0.5 a step while there is one a CU, 0.8 when there are two, and
//     for every further two;
//   128-row tiles: 5.0 + 0.7 and 1.23 alike.
// None is faster than reading the experts' weights at 5.9 TB/s, which the first comes
// nearest to.  Measured against each other (rows, 64, 128), us:
//   gate/up 64 experts, D 2048, F 1024, top-8: 1 token 4.8, 11.6, 15.4; 48 tokens 24.0,
//     25.0, 27.6; 512 tokens 39.9, 33.3, 35.9; 1000 tokens 68.7, 36.9, 35.9;
//   32 experts, D 4096, F 2048, top-4: 300 tokens 68.2, 51.7, 64.1;
//   24 experts, D 1152, F 640, top-3: 333 tokens 7.9, 8.9, 11.4; 800 tokens 13.2, 9.0,
//     11.4; 2000 tokens 22.7, 16.6, 14.4;
//   one segment, D 2048, F 1024: 64 rows 5.6, 11.9, 15.4; 2000 rows 19.4, 12.2, 15.7; 8000
//     rows 64.7, 28.1, 23.7.
// Below four steps the split has nothing to split: 2000 tokens on 8 experts, D 256, 8.7
// against 5.5 with the waves side by side.
enum Form { kRows1, kRows4, kTiles64, kTiles128 };

// The experts that have rows, and the row tiles of all.  The counts are known only to
// the device: an expert is taken to have none as often as chance has it, and past three
// quarters of a tile some need another.
double live_experts(int64_t rows, int n_experts) {
  return n_experts * -std::expm1(-static_cast<double>(rows) / n_experts);
}
double row_tiles(int64_t rows, int n_experts, int bm) {
  if (n_experts == 1) return static_cast<double>(ceil_div(rows, bm));
  const double n = live_experts(rows, n_experts), mean = rows / n;
  return n * (mean <= 0.75 * bm ? 1.0 : mean / bm + 0.5);
}

Form choose_form(int64_t rows, int n_experts, int kdim, int ncols, int cus) {
  const double steps = kdim / 128;
  const double n = live_experts(rows, n_experts);
  const double weights = n * ncols * kdim * (17.0 / 32.0) / 5.9e6;
  const double tiles32 = row_tiles(rows, n_experts, 32);
  const double by_rows = std::max(3.5 + tiles32 * (ncols / 64) * steps * 0.55e-3, weights * (0.9 + 0.1 * tiles32 / n));
  const auto by_tiles = [&](int bm, double start, double alone, double paired) {
    const double tiles = row_tiles(rows, n_experts, bm) * static_cast<double>(ceil_div(ncols, kTileN));
    const double step = tiles <= cus ? alone : paired * std::ceil(tiles / (2.0 * cus) - 0.02);
    return std::max(start + steps * step, 1.1 * weights);
  };
  const double by_64 = by_tiles(64, 4.2, 0.5, 0.8);
  const double by_128 = steps > 1 ? by_tiles(128, 5.0, 0.7, 1.23) : by_64 + 1.0;
  // (a grid holds 65535 tiles along y)
  if (by_rows <= std::min(by_64, by_128) && max_row_tiles(rows, n_experts) <= 65535)
    return steps < 4 ? kRows1 : kRows4;
  return by_64 <= by_128 ? kTiles64 : kTiles128;
}

template <bool GATE_UP, bool GATHER>
int launch_product(const char* what, const uint8_t* a, const uint8_t* a_exp, const uint8_t* b,
                   const uint8_t* b_exp, const int32_t* offsets, int n_experts, int64_t rows_cap, int kdim,
                   int ncols, uint8_t* c, uint8_t* c_exp, const int32_t* gather_src, int gather_k,
                   int gather_rows, hipStream_t s) {
  HMOE_REQUIRE(static_cast<int64_t>(kdim / 128) * ncols * 4 < (int64_t(1) << 31), "%s: operand too large", what);
  HMOE_REQUIRE((ceil_div(rows_cap, 64) + n_experts) * ceil_div(ncols, kTileN) <= (int64_t(1) << 30),
               "%s: too many tiles", what);
  int dev = 0, cus = 0;
  if (int rc = persistent_grid(what, s, &cus, &dev)) return rc;
  const Form form = choose_form(rows_cap, n_experts, kdim, ncols, cus);
  if (form == kTiles64 || form == kTiles128) {
    const auto launch = [&](auto BM) {
      constexpr int bm = decltype(BM)::value;
      static std::atomic<uint64_t> done{0};
      if (int rc = allow_lds(what, grouped_mxfp4_tiles<bm, GATE_UP, GATHER>, TileCfg<bm>::kLds, dev, &done)) return rc;
      hipLaunchKernelGGL((grouped_mxfp4_tiles<bm, GATE_UP, GATHER>), dim3(2 * cus), dim3(kTileThreads),
                         TileCfg<bm>::kLds, s, a, a_exp, b, b_exp, offsets, n_experts, kdim, ncols, c, c_exp,
                         gather_src, gather_k, gather_rows);
      return check_launch(what);
    };
    return form == kTiles64 ? launch(std::integral_constant<int, 64>{}) : launch(std::integral_constant<int, 128>{});
  }
  const unsigned m_tiles = static_cast<unsigned>(max_row_tiles(rows_cap, n_experts));
  if (form == kRows4)
    hipLaunchKernelGGL((grouped_mxfp4_rows<GATE_UP, GATHER, 4>), dim3(ncols / 64, m_tiles), dim3(256), 0, s, a, a_exp,
                       b, b_exp, offsets, n_experts, kdim, ncols, c, c_exp, gather_src, gather_k, gather_rows);
  else
    hipLaunchKernelGGL((grouped_mxfp4_rows<GATE_UP, GATHER, 1>),
                       dim3(static_cast<unsigned>(ceil_div(ncols, 256)), m_tiles), dim3(256), 0, s, a, a_exp, b, b_exp,
                       offsets, n_experts, kdim, ncols, c, c_exp, gather_src, gather_k, gather_rows);
  return check_launch(what);
}

}  // namespace
}  // namespace hmoe

extern "C" int64_t hmoe_grouped_mxfp4_form(int64_t rows_cap, int n_experts, int kdim, int ncols, int cus) {
  using namespace hmoe;
  if (rows_cap < 1 || rows_cap > kMaxRows || n_experts < 1 || n_experts > kMaxExperts || cus < 1 || kdim < 128 || kdim % 128 != 0 ||
      ncols < 128 || ncols % 128 != 0) {
    set_error("grouped_mxfp4_form: sizes that the products refuse");
    return -1;
  }
  return choose_form(rows_cap, n_experts, kdim, ncols, cus);
}

extern "C" int hmoe_grouped_gate_up_mxfp4(const uint8_t* xs_q, const uint8_t* xs_exp, const int32_t* offsets,
                                          int n_experts, int64_t rows_cap, int d_model, int d_ff,
                                          const uint8_t* w_packed, const uint8_t* w_exp, uint8_t* h_q,
                                          uint8_t* h_exp, hmoe_stream_t stream) {
  using namespace hmoe;
  const char* what = "grouped_gate_up_mxfp4";
  if (int rc = check_product(what, n_experts, rows_cap, d_model, d_ff)) return rc;
  if (rows_cap == 0) return HMOE_OK;
  HMOE_REQUIRE(xs_q && xs_exp && offsets && w_packed && w_exp && h_q && h_exp, "%s: null pointer argument", what);
  HMOE_REQUIRE_ALIGNED(what, 16, xs_q, w_packed, h_q);
  HMOE_REQUIRE_ALIGNED(what, 4, xs_exp, w_exp, h_exp);
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
  HMOE_REQUIRE_ALIGNED(what, 16, x_q, w_packed, h_q);
  HMOE_REQUIRE_ALIGNED(what, 4, x_exp, w_exp, h_exp);
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
  HMOE_REQUIRE_ALIGNED(what, 16, h_q, w_packed, ys);
  HMOE_REQUIRE_ALIGNED(what, 4, h_exp, w_exp);
  return launch_product<false, false>(what, h_q, h_exp, w_packed, w_exp, offsets, n_experts, rows_cap, d_ff,
                                      d_model, static_cast<uint8_t*>(ys), nullptr, nullptr, 1, 1,
                                      static_cast<hipStream_t>(stream));
}
