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
#include <type_traits>

#include "grouped_tiles.h"
#include "quant_mxfp4.h"

namespace hmoe {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

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

// Epilogues.  Lane L of an accumulator holds row L % 32 of A's fragment and columns 8 q
// + 4 (L / 32) + 0..3 (q = 0..3) of B's.  Stores go through a buffer whose range ends
// at the segment's last row.
//
// h of 32 columns (gate in g, up in u), one scale block of the row: its exponent, and in
// w[0] this lane's halves of dwords 0 and 1 of the row's 16 bytes of codes, in w[1] of
// dwords 2 and 3.
__device__ __forceinline__ uint32_t quantise_h(const f32x16& g, const f32x16& u, uint32_t (&w)[2]) {
  float h[16];
  float amax = 0.0f;
#pragma unroll
  for (int k = 0; k < 16; k += 2) {
    h[k] = swiglu_f32(g[k], u[k]);
    h[k + 1] = swiglu_f32(g[k + 1], u[k + 1]);
    // (NaN where either is)
    amax = __builtin_elementwise_maximum(__builtin_elementwise_maximum(amax, __builtin_fabsf(h[k])),
                                         __builtin_fabsf(h[k + 1]));
  }
  // lanes L and L + 32 hold the row's other values
  const uint32_t am = __float_as_uint(amax);
  const auto sw = __builtin_amdgcn_permlane32_swap(am, am, false, false);
  const uint32_t e = mxfp4_exponent(sw[0] > sw[1] ? sw[0] : sw[1]);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = h[8 * j + k];
    w[j] = mxfp4_codes8(v, e);
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
    uint8_t* __restrict__ C, uint8_t* __restrict__ c_exp, const int32_t* __restrict__ gather_src,
    Divisor gather_k, int gather_rows) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int frow = lane & 31, half = lane >> 5;
  RowTile t;
  if (!find_row_tile(offsets, n_experts, 32, blockIdx.y, t)) return;
  const int n0 = SPLIT == 1 ? (blockIdx.x * 4 + wave) * 64 : blockIdx.x * 64;
  if (n0 >= ncols) return;  // (SPLIT 1 only: no barrier follows there)
  int src = t.row0 + (frow < t.rows ? frow : t.rows - 1);  // rows past the segment repeat its last one
  if (GATHER) src = token_of(gather_src[src], gather_k, gather_rows);
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
// Workgroups of four waves, two (BM 128) or three (BM 64) a CU, each looping over BM x 256
// tiles: while one is in its epilogue (the SwiGLU's exponentials and reciprocals alone take
// a quarter of the products' time), switches tiles or waits at its barrier, the others'
// products run.  A wave has all of the tile's rows and 64 of its columns, so B's fragments
// are read by one wave only and go from memory straight into registers, 1 KB an
// instruction, each loaded for the next step as soon as its products are issued.  A goes
// through LDS (buffer_load ... lds), two stages of 256 values = 128 bytes of every row, the
// next stage's loads issued behind the one barrier of a step: whole lines (64-byte pieces
// of rows come at 31 bytes a cycle and CU, 128-byte ones at 55), and 16-byte chunk c of row
// r sits at c ^ swz128(r), so that 16 lanes of a fragment read cover all banks.  A's
// exponents, 16 bytes of every row, come for two steps at once into one of two regions.
// Where K is an odd multiple of 128 the last step is half a one.  The last column tile may
// be 128 columns wide: waves 2 and 3 then load and compute the others' again and store
// nothing.
//
// Of two waves on a SIMD the older one's products go first, so that its workgroup took 23
// thousand cycles a tile and the other 32, which then ended alone: they take turns by tile
// (gate/up below 298 -> 285 us, down 172 -> 165; with 64 rows, taken where a workgroup has
// few tiles, 512 tokens 28.8 -> 32.0, and not done).
//
// Gate/up of 131072 rows, D 2048, F 1024 (1.1 TFLOP) takes 277 to 285 us; down 157 to 165
// us launched again and again and 203 behind the gate/up product (an output of 537 MB waits
// for what lies written in the caches).  With these operands the matrix cores alone, fed from
// registers, run at 1.65 GHz and 6.5 PFLOP/s (170 us) at the package's power limit; with
// operands of zeros, at 2.4 GHz, the same launches take 205 and 119 us (the products alone
// 113 and 57).  Power is not all: the matrix cores are busy in 54 % of gate/up's cycles (1.75
// GHz) and 34 % of down's behind it (1.96 GHz).  A tile ends in a phase without a product
// (the SwiGLU and quantisation; packing and stores), every 8 steps of K 2048 and every 4 of
// K 1024, which only another workgroup's products cover.  Gate/up with zeros takes 170 us
// with the products taken out, 161 with all loads and reads taken out instead, 198 with
// every load a hit of the first cache.
// Measured and not taken (us; gate/up and down, before the turns 300 and 170): B through LDS
// too (2 x 2 waves, steps of 128 values, three stages) 326 and 187, an LDS and half lines of
// A that kept pace with the products at best; one workgroup of eight waves on 128 x 512 301
// and 176; loads and reads issued one by one behind each product, A two steps ahead, 293
// and 173; the barrier ahead of a step's last products 290 and 169; the next tile brought
// into L2 during the epilogue 306 and 175; row-tile groups of 2, 4 and 16 the same as of 8;
// h stored from the accumulators, 16 bytes of a row at a time, 295.
constexpr int kTileThreads = 256;
template <int BM, bool GATE_UP>
struct TileCfg {
  static constexpr int kA = BM * 128, kExA = BM * 16;  // a stage, a region of exponents
  static constexpr int kOut = GATE_UP ? BM * 68 : 4 * 4096;  // h's codes and exponents; ys, 4 KB a wave
  static constexpr int kLds = 2 * (kA + kExA) + kOut;
  static constexpr int kFR = BM / 32;             // row fragments; DMA instructions a wave and step
  static constexpr int kPerCu = BM == 64 ? 3 : 2;
  static_assert(kPerCu * kLds <= 160 * 1024, "workgroups a CU");
};

// Of a CU's two workgroups one goes first.
__device__ __forceinline__ void take_turn(int turn) {
  if (turn == 0) __builtin_amdgcn_s_setprio(0);
  else __builtin_amdgcn_s_setprio(1);
}

template <int BM, bool GATE_UP, bool GATHER>
__global__ __launch_bounds__(kTileThreads, BM == 64 ? 3 : 2) void grouped_mxfp4_tiles(
    const uint8_t* __restrict__ A, const uint8_t* __restrict__ a_exp, const uint8_t* __restrict__ B,
    const uint8_t* __restrict__ b_exp, const int32_t* __restrict__ offsets, int n_experts, int kdim, int ncols,
    uint8_t* __restrict__ C, uint8_t* __restrict__ c_exp, const int32_t* __restrict__ gather_src,
    Divisor gather_k, int gather_rows, Divisor by_cols, Divisor by_group) {
  typedef TileCfg<BM, GATE_UP> Cfg;
  constexpr int kFR = Cfg::kFR;
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
  const int nb = (ks + 1) / 2;  // steps of 256 values
  const int row_bytes = kdim / 2, ex_bytes = kdim / 32;

  // ---- load side -----------------------------------------------------------------
  // A: instruction j of wave w fills rows (BM / 4) w + 8 j + lane / 8, chunk (lane & 7) ^
  // swz128(row) of the row's 128 bytes.
  TileCursor<BM> ld;
  ld.find(offsets, n_experts, divide(first, by_cols));
  TileCursor<BM> cur = ld, nx = ld;
  const int a_row = (BM / 4) * wave + (lane >> 3);
  __amdgpu_buffer_rsrc_t a_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(A), 0,
                                                                    GATHER ? gather_rows * row_bytes : 0, kBufferWord3);
  __amdgpu_buffer_rsrc_t ae_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a_exp), 0,
                                                                     GATHER ? gather_rows * ex_bytes : 0, kBufferWord3);
  __amdgpu_buffer_rsrc_t b_rsrc = a_rsrc, be_rsrc = a_rsrc;
  uint32_t a_voff[kFR], ae_voff = 0;
  const int b_col = (kdim / 64) * 1024;  // bytes of 32 columns
  int b_wave = 0, be_wave = 0;           // where this wave's columns begin
  const bool ex_a = wave < BM / 64;      // the waves that bring A's exponents
  int ld_kb = 0, ld_t = first, ld_region = 1, ld_stage = 0;
  int32_t pf_src[kFR], pf_ex = 0;  // GATHER: sources of this lane's rows of the tile after, nx
  auto a_byte = [&](int j) __attribute__((always_inline)) {
    return static_cast<uint32_t>(((lane & 7) ^ swz128(8 * j + (lane >> 3))) * 16);
  };
  auto fetch_src = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kFR; ++j) {
      const int r = a_row + 8 * j;
      pf_src[j] = gather_src[nx.row0 + (r < nx.rows ? r : nx.rows - 1)];
    }
    const int r = 64 * wave + lane;
    pf_ex = gather_src[nx.row0 + (r < nx.rows ? r : nx.rows - 1)];
  };
  auto token = [&](int32_t slot) __attribute__((always_inline)) {
    return static_cast<uint32_t>(token_of(slot, gather_k, gather_rows));
  };
  // Tile ld_t becomes the one that is loaded.
  auto set_load_tile = [&]() __attribute__((always_inline)) {
    if (GATHER) {
      ld = nx;
#pragma unroll
      for (int j = 0; j < kFR; ++j) a_voff[j] = token(pf_src[j]) * static_cast<uint32_t>(row_bytes) + a_byte(j);
      ae_voff = token(pf_ex) * static_cast<uint32_t>(ex_bytes);
      if (ld_t + per_xcd < hi) nx.move(offsets, ld_t + per_xcd, n_tiles_n, by_cols, by_group);
      fetch_src();  // (on every path: a load that may not be issued is waited for at once)
    } else {
      ld.move(offsets, ld_t, n_tiles_n, by_cols, by_group);
      // rows past the segment repeat its last one; their results are not stored
      a_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(A + static_cast<int64_t>(ld.row0) * row_bytes),
                                                 0, ld.rows * row_bytes, kBufferWord3);
      ae_rsrc = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint8_t*>(a_exp + static_cast<int64_t>(ld.row0) * ex_bytes), 0, ld.rows * ex_bytes, kBufferWord3);
#pragma unroll
      for (int j = 0; j < kFR; ++j) {
        const int r = a_row + 8 * j;
        a_voff[j] = static_cast<uint32_t>((r < ld.rows ? r : ld.rows - 1) * row_bytes) + a_byte(j);
      }
      const int r = 64 * wave + lane;
      ae_voff = static_cast<uint32_t>((r < ld.rows ? r : ld.rows - 1) * ex_bytes);
    }
    const int64_t block = static_cast<int64_t>(ld.e) * (ncols / 32) + ld.n0 / 32;
    const int width = ncols - ld.n0 < kTileN ? ncols - ld.n0 : kTileN;
    const int part = 64 * wave < width ? wave : wave - 2;  // (a tile of 128 columns: waves 0 and 1 again)
    b_wave = part * 2 * b_col;
    be_wave = part * 256;
    b_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(B + block * b_col), 0, width * row_bytes,
                                               kBufferWord3);
    be_rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(b_exp + (static_cast<int64_t>(ld.e) * ks * ncols + ld.n0) * 4), 0,
        ((ks - 1) * ncols + width) * 4, kBufferWord3);
    ld_kb = 0;
  };
  auto issue_a = [&]() __attribute__((always_inline)) {
    if ((ld_kb & 1) == 0) {
      ld_region ^= 1;
      // (what it reads past a row's end is not used; past the buffer it is not read)
      if (ex_a)
        dma16(ae_rsrc, smem + 2 * Cfg::kA + ld_region * Cfg::kExA + wave * 1024,
              ae_voff + static_cast<uint32_t>(ld_kb * 8));
    }
#pragma unroll
    for (int j = 0; j < kFR; ++j)
      dma16(a_rsrc, smem + ld_stage * Cfg::kA + (wave * kFR + j) * 1024, a_voff[j] + static_cast<uint32_t>(ld_kb * 128));
    ld_stage ^= 1;
    fence();  // (the waits count B's loads behind these)
  };
  u32x4 fb[4][2];
  uint32_t eb[2][2];
  // B of the step that is loaded.  (Past the tile's last value: the last again, not used.)
  auto load_b = [&](int q) __attribute__((always_inline)) {
    const int k64 = 4 * ld_kb + q < 2 * ks ? 4 * ld_kb + q : 2 * ks - 1;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      fb[q][j] = __builtin_amdgcn_raw_buffer_load_b128(b_rsrc, lane * 16, b_wave + j * b_col + k64 * 1024, 0);
  };
  auto load_eb = [&](int t) __attribute__((always_inline)) {
    const int k128 = 2 * ld_kb + t < ks ? 2 * ld_kb + t : ks - 1;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      eb[t][j] = __builtin_amdgcn_raw_buffer_load_b32(be_rsrc, (lane & 31) * 4, be_wave + j * 128 + k128 * ncols * 4, 0);
  };

  // ---- compute side ----------------------------------------------------------------
  // Wave w: all rows and columns 64 w .. of the tile.
  const int frow = lane & 31, half = lane >> 5;
  const int fsw = swz128(frow);
  f32x16 acc[kFR][2];
  int stage = 0, region = 1;
  constexpr int kNewer = 12;  // loads of B and its exponents in a step, behind A's

  // One step: 64 nq values of this tile, the loads of the next step behind them.
  auto step = [&](int kb, auto NQ) __attribute__((always_inline)) {
    constexpr int nq = decltype(NQ)::value;
    // this wave's loads of A have landed; after the barrier every wave's have, and every
    // wave is done with the step before, whose stage the next loads take
    wait_vm_lgkm0<kNewer>();
    __builtin_amdgcn_s_barrier();
    fence();
    // on to the next step (after the last tile's last one: it again)
    if (ld_kb + 1 < nb) {
      ++ld_kb;
    } else if (ld_t + per_xcd < hi) {
      ld_t += per_xcd;
      set_load_tile();
    }
    issue_a();
    if ((kb & 1) == 0) region ^= 1;
    const uint8_t* st = smem + stage * Cfg::kA + frow * 128;
    const uint8_t* se = smem + 2 * Cfg::kA + region * Cfg::kExA + frow * 16 + (kb & 1) * 8;
    u32x2_t exw[kFR];
    u32x4 fa[2][kFR];
    auto read_a = [&](int q) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kFR; ++i)
        fa[q & 1][i] = *reinterpret_cast<const u32x4*>(st + i * 4096 + (((2 * q + half) ^ fsw) * 16));
    };
    read_a(0);
#pragma unroll
    for (int i = 0; i < kFR; ++i) exw[i] = *reinterpret_cast<const u32x2_t*>(se + i * 512);
    int ebs[2];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (q < nq) {
        // (kept ahead of the products, or each fragment is waited for)
        if (q + 1 < nq) read_a(q + 1);
        __builtin_amdgcn_sched_barrier(0);
        int ea[kFR];
#pragma unroll
        for (int i = 0; i < kFR; ++i) ea[i] = static_cast<int>(exw[i][q >> 1] >> (8 * half));
        if ((q & 1) == 0) {  // (then the words themselves are free)
#pragma unroll
          for (int j = 0; j < 2; ++j) ebs[j] = static_cast<int>(eb[q >> 1][j] >> (8 * half));
        }
        if (q == 0 && kb == 0) {  // (zeros as an operand, not written first)
          const f32x16 zero = {};
#pragma unroll
          for (int i = 0; i < kFR; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = mfma_fp4<0>(fb[0][j], fa[0][i], zero, ebs[j], ea[i]);
        } else {
#pragma unroll
          for (int i = 0; i < kFR; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              acc[i][j] = (q & 1) ? mfma_fp4<2>(fb[q][j], fa[q & 1][i], acc[i][j], ebs[j], ea[i])
                                  : mfma_fp4<0>(fb[q][j], fa[q & 1][i], acc[i][j], ebs[j], ea[i]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      load_b(q);
      if ((q & 1) == 0) load_eb(q >> 1);
      fence();
    }
#pragma unroll
    for (int i = 0; i < kFR; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) use_here(acc[i][j]);
    stage ^= 1;
  };

  if (GATHER) {
    nx.move(offsets, first, n_tiles_n, by_cols, by_group);
    fetch_src();
  }
  set_load_tile();
  issue_a();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    load_b(q);
    if ((q & 1) == 0) load_eb(q >> 1);
  }
  fence();
  int turn = blockIdx.x < gridDim.x / 2;  // (workgroups i and i + gridDim / 2 share a CU)
  for (int t = first; t < hi; t += per_xcd) {
    int kb = 0;
    if (BM == 128) take_turn(turn ^= 1);
    for (; 2 * kb + 1 < ks; ++kb) step(kb, std::integral_constant<int, 4>{});
    if (2 * kb < ks) step(kb, std::integral_constant<int, 2>{});  // 128 values
    cur.move(offsets, t, n_tiles_n, by_cols, by_group);
    const int64_t r0 = cur.row0;
    if constexpr (GATE_UP) {
      const int d_ff = ncols / 2;
      const __amdgpu_buffer_rsrc_t q_out =
          __builtin_amdgcn_make_buffer_rsrc(C + r0 * (d_ff / 2), 0, cur.rows * (d_ff / 2), kBufferWord3);
      const __amdgpu_buffer_rsrc_t e_out =
          __builtin_amdgcn_make_buffer_rsrc(c_exp + r0 * (d_ff / 32), 0, cur.rows * (d_ff / 32), kBufferWord3);
      // 64 bytes of every row's codes and four exponents are put together in LDS (each wave
      // has 16 and one of them)
      uint8_t* const codes = smem + 2 * (Cfg::kA + Cfg::kExA);
      uint8_t* const exps = codes + BM * 64;
#pragma unroll
      for (int i = 0; i < kFR; ++i) {
        uint32_t w[2];
        const uint32_t e = quantise_h(acc[i][0], acc[i][1], w);
        const auto sw = __builtin_amdgcn_permlane32_swap(w[0], w[1], false, false);
        *reinterpret_cast<u32x2_t*>(codes + (32 * i + frow) * 64 + wave * 16 + half * 8) = join_codes(sw[0], sw[1]);
        if (half == 0) exps[(32 * i + frow) * 4 + wave] = static_cast<uint8_t>(e);
      }
      fence();  // (the wait and the barrier are no memory accesses to the compiler)
      wait_lgkm0();
      __builtin_amdgcn_s_barrier();
      fence();
      const int width = ncols - cur.n0 < kTileN ? ncols - cur.n0 : kTileN;
#pragma unroll
      for (int m = 0; m < BM / 64; ++m) {
        const int row = (BM / 4) * wave + 16 * m + (lane >> 2);
        const u32x4 v = *reinterpret_cast<const u32x4*>(codes + row * 64 + (lane & 3) * 16);
        if ((lane & 3) * 64 < width)
          __builtin_amdgcn_raw_buffer_store_b128(v, q_out, (row * d_ff + cur.n0 / 2) / 2 + (lane & 3) * 16, 0, 0);
      }
      if (lane < BM / 4) {
        const int row = (BM / 4) * wave + lane;
        const uint32_t v = *reinterpret_cast<const uint32_t*>(exps + row * 4);
        const int off = row * (d_ff / 32) + cur.n0 / 64;
        if (width == kTileN) __builtin_amdgcn_raw_buffer_store_b32(v, e_out, off, 0, 0);
        else __builtin_amdgcn_raw_buffer_store_b16(static_cast<uint16_t>(v), e_out, off, 0, 0);
      }
    } else {
      const __amdgpu_buffer_rsrc_t out =
          __builtin_amdgcn_make_buffer_rsrc(C + r0 * ncols * 2, 0, cur.rows * ncols * 2, kBufferWord3);
      const bool mine = cur.n0 + wave * 64 < ncols;  // uniform per wave
      uint8_t* const lds = smem + 2 * (Cfg::kA + Cfg::kExA) + wave * 4096;
#pragma unroll
      for (int i = 0; i < kFR; ++i)
        if (mine) store_y_blocks(acc[i][0], acc[i][1], lds, out, 32 * i, cur.n0 + wave * 64, ncols, lane);
    }
    fence();  // (this tile's reads of LDS stay ahead of the next step's barrier)
  }
  // nothing may still be writing into LDS when the workgroup ends
  __builtin_amdgcn_s_waitcnt(0);
}

// The checks that the products share.
int check_product(const char* what, int n_experts, int64_t rows_cap, int d_model, int d_ff) {
  HMOE_REQUIRE(n_experts >= 1 && n_experts <= kMaxExperts, "%s: n_experts must be in [1, %d] (got %d)", what,
               kMaxExperts, n_experts);
  // (2^30: a tile's rows and the tiles that a workgroup steps over are added in 32 bits)
  HMOE_REQUIRE(rows_cap >= 0 && rows_cap <= kMaxRows, "%s: rows_cap must be in [0, 2^30]", what);
  HMOE_REQUIRE_CODE(d_model >= 128 && d_model % 128 == 0 && d_model <= kMaxDim, HMOE_ERR_UNSUPPORTED,
                    "%s: d_model must be a multiple of 128 up to 2^20 (got %d)", what, d_model);
  HMOE_REQUIRE_CODE(d_ff >= 128 && d_ff % 128 == 0 && d_ff <= kMaxDim, HMOE_ERR_UNSUPPORTED,
                    "%s: d_ff must be a multiple of 128 up to 2^20 (got %d)", what, d_ff);
  return HMOE_OK;
}

// What a launch cannot count in 32 bits, beyond the sizes that check_product looks at: an
// expert's exponents in bytes, the tiles of the smaller tile form.
const char* too_large(int64_t rows_cap, int n_experts, int kdim, int ncols) {
  if (static_cast<int64_t>(kdim / 128) * ncols * 4 >= (int64_t(1) << 31)) return "operand too large";
  if ((ceil_div(rows_cap, 64) + n_experts) * ceil_div(ncols, kTileN) > (int64_t(1) << 30)) return "too many tiles";
  return nullptr;
}

// Which kernel a product takes: the one with the least estimated time, from measured
// rates (MI355X, us, `steps` = K / 128):
//   rows: 3.5, and 0.55 ns for every 32 rows x 64 columns x 128 values (0.35 unsplit); or the
//     experts' weights at 5.9 TB/s and, for every 64 columns, the rows at 8;
//   64-row tiles, three a CU at a time: 3.6, and 0.34 a step for each that a CU has, 0.36 for
//     one alone; or the weights and 1.5;
//   128-row tiles, two a CU: 4.2, 0.545 and 0.52.
// Measured against each other (rows, 64, 128), us:
//   gate/up 64 experts, D 2048, F 1024, top-8: 1 token 5.6, 8.7, 11.8; 8 tokens 14.8, 17.8,
//     20.4; 64 tokens 24.5, 23.5, 25.3; 128 tokens 26.4, 24.3, 26.0; 1000 tokens 63, 32.0,
//     37; 1500 tokens 89, 40, 46; 4000 tokens 213, 86, 80; 16384 tokens 792, 330, 285;
//   32 experts, D 4096, F 2048, top-4: 300 tokens 69, 49.8, 59.6; 2000 tokens 238, 111, 91;
//   24 experts, D 1152, F 640, top-3: 100 tokens 5.5, 7.2, 9.2; 333 tokens 8.0, 7.2, 9.3;
//     4000 tokens 34, 17.1, 22;
//   one segment, D 2048, F 1024: 200 rows 5.8, 8.9, 11.8; 1000 rows 10.0, 9.0, 12.0; 8000
//     rows 54, 22.9, 21.5.
// Rows split the reduction where there are few waves or it is long; below 16 steps waves
// side by side that fill the chip are faster: down of 64 experts (8 steps), 32 tokens 12.2
// against 13.3, of 128 experts, D 1024, F 512 (4 steps), 30 tokens 5.0 against 6.1.  Below
// four steps there is nothing to split.
// The rule does not always choose the fastest (forms 0, 1, 2, 3 measured, us): a split that is
// taken below 4 waves a CU and charged 0.55 lets down of 64 experts, D 2048, F 1024, go to 64-row
// tiles at 4 and 5 tokens (4.4, 4.5, 6.0, 7.6) and of 128 experts, D 2048, F 768, at 3 and 4
// (4.4, 4.4, 5.8, 7.2; 5.1, 5.0, 5.8, 7.2); where the weights bound both sides, gate/up of 128
// experts, D 4096, F 1536, 16 tokens goes there too (84.9, 75.1, 79.9, 80.7).
enum Form { kRows1, kRows4, kTiles64, kTiles128 };

Form choose_form(int64_t rows, int n_experts, int kdim, int ncols, int cus) {
  const double steps = kdim / 128;
  const double n = live_experts(rows, n_experts);
  const double weights = n * ncols * kdim * (17.0 / 32.0) / 5.9e6;
  const double tiles32 = row_tiles(rows, n_experts, 32);
  const double re_read = static_cast<double>(rows) * (ncols / 64) * (kdim / 2) / 8e6;
  const double waves = tiles32 * (ncols / 64);
  const bool split = steps >= 16 || (steps >= 4 && waves < 4.0 * cus);
  const double by_rows = std::max(3.5 + waves * steps * (split ? 0.55e-3 : 0.35e-3), weights + re_read);
  const auto by_tiles = [&](int bm, int per_cu, double start, double alone, double busy) {
    const double tiles = row_tiles(rows, n_experts, bm) * static_cast<double>(ceil_div(ncols, kTileN));
    const double whole = std::floor(tiles / (per_cu * cus)), rest = tiles - whole * per_cu * cus;
    const double last = rest < 1.0 ? 0.0 : std::max(alone, busy * std::ceil(rest / cus - 0.02));
    return std::max(start + steps * (whole * per_cu * busy + last), weights + 1.5);
  };
  const double by_64 = by_tiles(64, TileCfg<64, true>::kPerCu, 3.6, 0.36, 0.34);
  const double by_128 = by_tiles(128, TileCfg<128, true>::kPerCu, 4.2, 0.52, 0.545);
  // (a grid holds 65535 tiles along y)
  if (by_rows <= std::min(by_64, by_128) && max_row_tiles(rows, n_experts) <= 65535)
    return split ? kRows4 : kRows1;
  return 0.92 * by_64 <= by_128 ? kTiles64 : kTiles128;  // (the counts are estimates: 64 rows end more evenly)
}

template <bool GATE_UP, bool GATHER>
int launch_product(const char* what, const uint8_t* a, const uint8_t* a_exp, const uint8_t* b,
                   const uint8_t* b_exp, const int32_t* offsets, int n_experts, int64_t rows_cap, int kdim,
                   int ncols, uint8_t* c, uint8_t* c_exp, const int32_t* gather_src, int gather_k,
                   int gather_rows, hipStream_t s) {
  const Divisor by_k = divisor(gather_k);
  const char* limit = too_large(rows_cap, n_experts, kdim, ncols);
  HMOE_REQUIRE(limit == nullptr, "%s: %s", what, limit);
  int dev = 0, cus = 0;
  if (int rc = persistent_grid(what, s, &cus, &dev)) return rc;
  const Form form = choose_form(rows_cap, n_experts, kdim, ncols, cus);
  if (form == kTiles64 || form == kTiles128) {
    const auto launch = [&](auto BM) {
      constexpr int bm = decltype(BM)::value;
      constexpr int lds = TileCfg<bm, GATE_UP>::kLds, per_cu = TileCfg<bm, GATE_UP>::kPerCu;
      const int n_tiles_n = static_cast<int>(ceil_div(ncols, kTileN));
      const Divisor by_cols = divisor(n_tiles_n), by_group = divisor(kTileGroup * n_tiles_n);
      static std::atomic<uint64_t> done{0};
      if (int rc = allow_lds(what, grouped_mxfp4_tiles<bm, GATE_UP, GATHER>, lds, dev, &done)) return rc;
      hipLaunchKernelGGL((grouped_mxfp4_tiles<bm, GATE_UP, GATHER>), dim3(per_cu * cus), dim3(kTileThreads),
                         lds, s, a, a_exp, b, b_exp, offsets, n_experts, kdim, ncols, c, c_exp,
                         gather_src, by_k, gather_rows, by_cols, by_group);
      return check_launch(what);
    };
    return form == kTiles64 ? launch(std::integral_constant<int, 64>{}) : launch(std::integral_constant<int, 128>{});
  }
  const unsigned m_tiles = static_cast<unsigned>(max_row_tiles(rows_cap, n_experts));
  if (form == kRows4)
    hipLaunchKernelGGL((grouped_mxfp4_rows<GATE_UP, GATHER, 4>), dim3(ncols / 64, m_tiles), dim3(256), 0, s, a, a_exp,
                       b, b_exp, offsets, n_experts, kdim, ncols, c, c_exp, gather_src, by_k, gather_rows);
  else
    hipLaunchKernelGGL((grouped_mxfp4_rows<GATE_UP, GATHER, 1>),
                       dim3(static_cast<unsigned>(ceil_div(ncols, 256)), m_tiles), dim3(256), 0, s, a, a_exp, b, b_exp,
                       offsets, n_experts, kdim, ncols, c, c_exp, gather_src, by_k, gather_rows);
  return check_launch(what);
}

}  // namespace
}  // namespace hmoe

extern "C" int64_t hmoe_grouped_mxfp4_form(int64_t rows_cap, int n_experts, int kdim, int ncols, int cus) {
  using namespace hmoe;
  if (rows_cap < 1 || rows_cap > kMaxRows || n_experts < 1 || n_experts > kMaxExperts || cus < 1 || kdim < 128 ||
      kdim % 128 != 0 || kdim > kMaxDim || ncols < 128 || ncols % 128 != 0 || ncols > 2 * kMaxDim ||
      too_large(rows_cap, n_experts, kdim, ncols) != nullptr) {
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
