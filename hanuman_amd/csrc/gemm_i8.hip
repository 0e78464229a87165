// Grouped products of int8 rows with int8 expert weights (model/moe.py:67-74 on 8-bit
// operands; the reference has no such path):
//
//   C[r, n] = a_scale[r] b_scale_e[n] sum_k A[r, k] B_e[n, k]   for rows r of expert e's segment
//
// on v_mfma_i32_32x32x32_i8.  The sums are exact: 32768 products of at most 2^14 stay below
// 2^31.  They are rounded to float32 once, then come the two scales, and for gate/up the
// SwiGLU, all in float32; h and ys are rounded to bf16 once.
//
// The operand keeps a lane's 16 bytes of a fragment together: lane 32 h + r of block (p /
// 32, k / 32) has the 16 codes of row r from column 16 h on, so a fragment is one 1 KB run
// of memory.  (Which of the instruction's 32 products a value takes part in does not matter,
// as long as both operands agree.)
#include <type_traits>

#include "grouped_tiles.h"
#include "quant_mxfp4.h"
#include "rows.h"

namespace hmoe {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ i32x16 mfma_i8(const u32x4& b, const u32x4& a, const i32x16& c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, b), __builtin_bit_cast(i32x4, a), c, 0, 0, 0);
}

// Sums of 32 columns to values: `cols` are the columns' scales.  Lane L holds row L % 32 and
// columns 8 q + 4 (L / 32) + 0..3 (q = 0..3).
__device__ __forceinline__ f32x16 scaled(const i32x16& acc, const float* cols, float row, int half) {
  f32x16 y;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const f32x4 c = *reinterpret_cast<const f32x4*>(cols + 8 * q + 4 * half);
#pragma unroll
    for (int i = 0; i < 4; ++i) y[4 * q + i] = static_cast<float>(acc[4 * q + i]) * c[i] * row;
  }
  return y;
}
__device__ __forceinline__ f32x16 swiglu16(const f32x16& g, const f32x16& u) {
  f32x16 h;
#pragma unroll
  for (int i = 0; i < 16; ++i) h[i] = swiglu_f32(g[i], u[i]);
  return h;
}

// ---- few rows ---------------------------------------------------------------------
// 32 rows x 64 columns a wave, operands straight from memory into registers: with few
// rows an expert every weight is used once or twice, and a fragment is one run of 1 KB.
// A workgroup is four waves: side by side (SPLIT 1), or on a quarter of the reduction
// each, joined in LDS (SPLIT 4; the sums are exact, so the order does not matter).  Bound by
// the latency of a wave's chain of loads, then by the weights' bytes: one token on 64 experts,
// top-8, D 2048, F 1024 (34 and 17 MB of weights) 9.8 us gate/up and 6.8 down, split (13.4
// gate/up side by side).
template <bool GATE_UP, bool GATHER, int SPLIT>
__global__ __launch_bounds__(256) void grouped_i8_rows(
    const int8_t* __restrict__ A, const float* __restrict__ a_scale, const int8_t* __restrict__ B,
    const float* __restrict__ b_scale, const int32_t* __restrict__ offsets, int n_experts, int kdim, int ncols,
    uint16_t* __restrict__ C, const int32_t* __restrict__ gather_src, Divisor gather_k, int gather_rows) {
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
  const int8_t* a = A + static_cast<int64_t>(src) * kdim + half * 16;
  const int64_t frag = (static_cast<int64_t>(t.e) * (ncols / 32) + n0 / 32) * (kdim / 32);
  const int8_t* b0 = B + frag * 1024 + lane * 16;
  const int8_t* b1 = b0 + static_cast<int64_t>(kdim / 32) * 1024;
  const float row_scale = a_scale[src];
  i32x16 acc0 = {}, acc1 = {};
  struct Group {
    u32x4 fa[4], f0[4], f1[4];
  };
  auto load = [&](Group& p, int k) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      p.fa[q] = *reinterpret_cast<const u32x4*>(a + k * 128 + q * 32);
      p.f0[q] = *reinterpret_cast<const u32x4*>(b0 + static_cast<int64_t>(k) * 4096 + q * 1024);
      p.f1[q] = *reinterpret_cast<const u32x4*>(b1 + static_cast<int64_t>(k) * 4096 + q * 1024);
    }
  };
  auto use = [&](const Group& p) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      acc0 = mfma_i8(p.f0[q], p.fa[q], acc0);
      acc1 = mfma_i8(p.f1[q], p.fa[q], acc1);
    }
  };
  int k = SPLIT == 1 ? 0 : groups * wave / SPLIT;
  const int end = SPLIT == 1 ? groups : groups * (wave + 1) / SPLIT;
  for (; k + 2 <= end; k += 2) {
    Group p[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) load(p[j], k + j);
#pragma unroll
    for (int j = 0; j < 2; ++j) use(p[j]);
  }
  for (; k < end; ++k) {
    Group p;
    load(p, k);
    use(p);
  }
  if constexpr (SPLIT > 1) {
    // wave 0 adds the others' sums
    __shared__ i32x4 part[SPLIT - 1][8][64];
    if (wave > 0) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        part[wave - 1][r][lane] = i32x4{acc0[4 * r], acc0[4 * r + 1], acc0[4 * r + 2], acc0[4 * r + 3]};
        part[wave - 1][4 + r][lane] = i32x4{acc1[4 * r], acc1[4 * r + 1], acc1[4 * r + 2], acc1[4 * r + 3]};
      }
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 0; w < SPLIT - 1; ++w)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const i32x4 p0 = part[w][r][lane], p1 = part[w][4 + r][lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc0[4 * r + i] += p0[i];
          acc1[4 * r + i] += p1[i];
        }
      }
  }
  const int64_t r0 = t.row0;
  const float* cs = b_scale + static_cast<int64_t>(t.e) * ncols + n0;
  const f32x16 y0 = scaled(acc0, cs, row_scale, half), y1 = scaled(acc1, cs + 32, row_scale, half);
  const int ldc = GATE_UP ? ncols / 2 : ncols;
  const __amdgpu_buffer_rsrc_t out =
      __builtin_amdgcn_make_buffer_rsrc(C + r0 * ldc, 0, t.rows * ldc * 2, kBufferWord3);
  if constexpr (GATE_UP) {
    store_y_block(swiglu16(y0, y1), out, frow, n0 / 2, ldc, half);
  } else {
    store_y_block(y0, out, frow, n0, ldc, half);
    store_y_block(y1, out, frow, n0 + 32, ldc, half);
  }
}

// ---- tiles for experts with many rows ------------------------------------------
// Workgroups of four waves, two (BM 128) or three (BM 64) a CU, each looping over BM x 256
// tiles: while one is in its epilogue, switches tiles or waits at its barrier, the others'
// products run.  A wave has all of the tile's rows and 64 of its columns, so B's fragments
// are read by one wave only and go from memory straight into registers, 1 KB an
// instruction, each loaded for the next step as soon as its products are issued.  A goes
// through LDS (buffer_load ... lds), two stages of 128 values of every row, the next
// stage's loads issued behind the one barrier of a step: whole lines, and 16-byte chunk c of
// row r sits at c ^ swz128(r), so that 16 lanes of a fragment read cover all banks.  A tile's
// scales come with its first step into one of two regions (from memory in the epilogue: 529 and
// 333 us against 506 and 269 below).  h is put together in LDS and leaves as 256 bytes of a row
// (1000 tokens on 64 experts 72 -> 64 us).  The last column tile may be 128 columns wide: waves 2
// and 3 then load and compute the others' again and store nothing.
//
// 131072 rows, D 2048, F 1024, gate/up and down: 500 and 270 us (2.2 and 2.0 POP/s; the matrix
// cores alone, from registers, 3.6, where the package's power takes the clock to 1.8 GHz; the
// vendor library's product of 16384 x 8192 x 8192 1.9).  They are busy in 63 % and 49 % of the
// cycles at 1.66 and 1.78 GHz, and a quarter of the lines that are asked for miss L2.  With operands
// of zeros (2.4 GHz) 394 and 202 us; every load a hit of L2 463 and 251; without the products 383 and 202:
// power, the loads' way and the epilogue (438 and 219 without it) share the time, none has all of
// it.  No faster: A three stages deep (508 and 275 against 517 and 280), steps in another order for
// each tile, row-tile groups of 1 to 32, two workgroups of 64 rows a CU, no turns.
constexpr int kTileThreads = 256;

template <int BM, bool GATE_UP>
struct TileCfg {
  static constexpr int kA = BM * 128;              // a stage
  static constexpr int kScales = BM * 4 + 1024;    // a tile's row and column scales
  // h of the whole tile, or 4 KB of ys a wave, on their way out
  static constexpr int kOut = GATE_UP ? BM * 256 : 4 * 4096;
  static constexpr int kLds = 2 * (kA + kScales) + kOut;
  static constexpr int kFR = BM / 32;              // row fragments; DMA instructions a wave and step
  static constexpr int kPerCu = BM == 64 ? 3 : 2;
  static_assert(kPerCu * kLds <= 160 * 1024, "workgroups a CU");
};

__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t r, uint8_t* dst, uint32_t voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)dst, 4, voff, 0, 0, 0);
}

__device__ __forceinline__ void use_here(const i32x16& v) { asm volatile("" ::"v"(v)); }

// Of a CU's two workgroups one goes first.
__device__ __forceinline__ void take_turn(int turn) {
  if (turn == 0) __builtin_amdgcn_s_setprio(0);
  else __builtin_amdgcn_s_setprio(1);
}

template <int BM, bool GATE_UP, bool GATHER>
__global__ __launch_bounds__(kTileThreads, BM == 64 ? 3 : 2) void grouped_i8_tiles(
    const int8_t* __restrict__ A, const float* __restrict__ a_scale, const int8_t* __restrict__ B,
    const float* __restrict__ b_scale, const int32_t* __restrict__ offsets, int n_experts, int kdim, int ncols,
    uint16_t* __restrict__ C, const int32_t* __restrict__ gather_src, Divisor gather_k, int gather_rows,
    Divisor by_cols, Divisor by_group) {
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
  const int ks = kdim / 128;  // steps
  const int row_bytes = kdim;

  // ---- load side -----------------------------------------------------------------
  // A: instruction j of wave w fills rows (BM / 4) w + 8 j + lane / 8, chunk (lane & 7) ^
  // swz128(row) of the row's 128 bytes.
  TileCursor<BM> ld;
  ld.find(offsets, n_experts, divide(first, by_cols));
  TileCursor<BM> cur = ld, nx = ld;
  const int a_row = (BM / 4) * wave + (lane >> 3);
  __amdgpu_buffer_rsrc_t a_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(A), 0,
                                                                    GATHER ? gather_rows * row_bytes : 0, kBufferWord3);
  __amdgpu_buffer_rsrc_t b_rsrc = a_rsrc;
  uint32_t a_voff[kFR];
  const int b_col = (kdim / 32) * 1024;  // bytes of 32 columns
  int b_wave = 0;                        // where this wave's columns begin
  __amdgpu_buffer_rsrc_t as_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a_scale), 0,
                                                                     GATHER ? gather_rows * 4 : 0, kBufferWord3);
  __amdgpu_buffer_rsrc_t bs_rsrc = a_rsrc;
  uint32_t as_voff = 0, bs_voff = 0;
  const bool row_scales = wave < BM / 64;  // the waves that bring the rows' scales
  int ld_kb = 0, ld_t = first, ld_stage = 0, ld_region = 1;
  int32_t pf_src[kFR], pf_scale = 0;  // GATHER: sources of this lane's rows of the tile after, nx
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
    pf_scale = gather_src[nx.row0 + (r < nx.rows ? r : nx.rows - 1)];
  };
  // Tile ld_t becomes the one that is loaded.
  auto set_load_tile = [&]() __attribute__((always_inline)) {
    if (GATHER) {
      ld = nx;
#pragma unroll
      for (int j = 0; j < kFR; ++j)
        a_voff[j] = static_cast<uint32_t>(token_of(pf_src[j], gather_k, gather_rows)) * static_cast<uint32_t>(row_bytes) +
                    a_byte(j);
      as_voff = static_cast<uint32_t>(token_of(pf_scale, gather_k, gather_rows)) * 4u;
      if (ld_t + per_xcd < hi) nx.move(offsets, ld_t + per_xcd, n_tiles_n, by_cols, by_group);
      fetch_src();  // (on every path: a load that may not be issued is waited for at once)
    } else {
      ld.move(offsets, ld_t, n_tiles_n, by_cols, by_group);
      // rows past the segment repeat its last one; their results are not stored
      a_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(A + static_cast<int64_t>(ld.row0) * row_bytes), 0,
                                                 ld.rows * row_bytes, kBufferWord3);
#pragma unroll
      for (int j = 0; j < kFR; ++j) {
        const int r = a_row + 8 * j;
        a_voff[j] = static_cast<uint32_t>((r < ld.rows ? r : ld.rows - 1) * row_bytes) + a_byte(j);
      }
      as_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a_scale + ld.row0), 0, ld.rows * 4, kBufferWord3);
      const int r = 64 * wave + lane;
      as_voff = static_cast<uint32_t>(r < ld.rows ? r : ld.rows - 1) * 4u;
    }
    const int64_t block = static_cast<int64_t>(ld.e) * (ncols / 32) + ld.n0 / 32;
    const int width = ncols - ld.n0 < kTileN ? ncols - ld.n0 : kTileN;
    const int part = 64 * wave < width ? wave : wave - 2;  // (a tile of 128 columns: waves 0 and 1 again)
    b_wave = part * 2 * b_col;
    b_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(B + block * b_col), 0, width * row_bytes,
                                               kBufferWord3);
    bs_rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<float*>(b_scale + static_cast<int64_t>(ld.e) * ncols + ld.n0), 0, width * 4, kBufferWord3);
    bs_voff = static_cast<uint32_t>(64 * part + lane) * 4u;
    ld_kb = 0;
  };
  auto issue_a = [&]() __attribute__((always_inline)) {
    if (ld_kb == 0) {  // the tile's scales, into the region that the tile before does not read
      ld_region ^= 1;
      uint8_t* const to = smem + 2 * Cfg::kA + ld_region * Cfg::kScales;
      if (row_scales) dma4(as_rsrc, to + wave * 256, as_voff);
      dma4(bs_rsrc, to + BM * 4 + wave * 256, bs_voff);
    }
#pragma unroll
    for (int j = 0; j < kFR; ++j)
      dma16(a_rsrc, smem + ld_stage * Cfg::kA + (wave * kFR + j) * 1024, a_voff[j] + static_cast<uint32_t>(ld_kb * 128));
    ld_stage ^= 1;
    fence();  // (the waits count B's loads behind these)
  };
  u32x4 fb[4][2];
  // B of the step that is loaded.
  auto load_b = [&](int q) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      fb[q][j] = __builtin_amdgcn_raw_buffer_load_b128(b_rsrc, lane * 16, b_wave + j * b_col + (4 * ld_kb + q) * 1024, 0);
  };

  // ---- compute side ----------------------------------------------------------------
  // Wave w: all rows and columns 64 w .. of the tile.
  const int frow = lane & 31, half = lane >> 5;
  const int fsw = swz128(frow);
  i32x16 acc[kFR][2];
  int stage = 0, region = 1;
  constexpr int kNewer = 8;  // loads of B in a step, behind A's

  // One step: 128 values of this tile, the loads of the next step behind them.
  auto step = [&](int kb) __attribute__((always_inline)) {
    // this wave's loads of A have landed; after the barrier every wave's have, and every
    // wave is done with the step before, whose stage the next loads take
    wait_vm_lgkm0<kNewer>();
    __builtin_amdgcn_s_barrier();
    fence();
    // on to the next step (after the last tile's last one: it again)
    if (ld_kb + 1 < ks) {
      ++ld_kb;
    } else if (ld_t + per_xcd < hi) {
      ld_t += per_xcd;
      set_load_tile();
    }
    issue_a();
    const uint8_t* st = smem + stage * Cfg::kA + frow * 128;
    u32x4 fa[2][kFR];
    auto read_a = [&](int q) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kFR; ++i)
        fa[q & 1][i] = *reinterpret_cast<const u32x4*>(st + i * 4096 + (((2 * q + half) ^ fsw) * 16));
    };
    read_a(0);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      // (kept ahead of the products, or each fragment is waited for)
      if (q + 1 < 4) read_a(q + 1);
      __builtin_amdgcn_sched_barrier(0);
      if (q == 0 && kb == 0) {  // (zeros as an operand, not written first)
        const i32x16 zero = {};
#pragma unroll
        for (int i = 0; i < kFR; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[i][j] = mfma_i8(fb[0][j], fa[0][i], zero);
      } else {
#pragma unroll
        for (int i = 0; i < kFR; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[i][j] = mfma_i8(fb[q][j], fa[q & 1][i], acc[i][j]);
      }
      __builtin_amdgcn_sched_barrier(0);
      load_b(q);
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
  for (int q = 0; q < 4; ++q) load_b(q);
  fence();
  int turn = blockIdx.x < gridDim.x / 2;  // (workgroups i and i + gridDim / 2 share a CU)
  for (int t = first; t < hi; t += per_xcd) {
    if (BM == 128) take_turn(turn ^= 1);
    for (int kb = 0; kb < ks; ++kb) step(kb);
    cur.move(offsets, t, n_tiles_n, by_cols, by_group);
    const int64_t r0 = cur.row0;
    const int ldc = GATE_UP ? ncols / 2 : ncols;
    const __amdgpu_buffer_rsrc_t out =
        __builtin_amdgcn_make_buffer_rsrc(C + r0 * ldc, 0, cur.rows * ldc * 2, kBufferWord3);
    const bool mine = cur.n0 + wave * 64 < ncols;  // uniform per wave
    region ^= 1;
    const float* const rs = reinterpret_cast<const float*>(smem + 2 * Cfg::kA + region * Cfg::kScales);
    const float* const cs = rs + BM + wave * 64;
    uint8_t* const stage_out = smem + 2 * (Cfg::kA + Cfg::kScales);
    if (mine) {
#pragma unroll
      for (int i = 0; i < kFR; ++i) {
        const float row_scale = rs[32 * i + frow];
        const f32x16 y0 = scaled(acc[i][0], cs, row_scale, half), y1 = scaled(acc[i][1], cs + 32, row_scale, half);
        if constexpr (GATE_UP) {
          // 256 bytes of every row are put together, chunk c of row r at c ^ (r & 15)
          u32x4 lo, hi;
          pack_y_block(swiglu16(y0, y1), lo, hi);
          uint8_t* const row = stage_out + (32 * i + frow) * 256;
          *reinterpret_cast<u32x4*>(row + (((4 * wave + half) ^ (frow & 15)) * 16)) = lo;
          *reinterpret_cast<u32x4*>(row + (((4 * wave + 2 + half) ^ (frow & 15)) * 16)) = hi;
        } else {
          store_y_blocks(y0, y1, stage_out + wave * 4096, out, 32 * i, cur.n0 + wave * 64, ldc, lane);
        }
      }
    }
    if constexpr (GATE_UP) {
      fence();  // (the wait and the barrier are no memory accesses to the compiler)
      wait_lgkm0();
      __builtin_amdgcn_s_barrier();
      fence();
      const int width = ncols - cur.n0 < kTileN ? ncols - cur.n0 : kTileN;
#pragma unroll
      for (int m = 0; m < BM / 16; ++m) {
        const int r = (BM / 4) * wave + 4 * m + (lane >> 4);
        const u32x4 v = *reinterpret_cast<const u32x4*>(stage_out + r * 256 + (((lane & 15) ^ (r & 15)) * 16));
        if ((lane & 15) * 16 < width)
          __builtin_amdgcn_raw_buffer_store_b128(v, out, (r * ldc + cur.n0 / 2) * 2 + (lane & 15) * 16, 0, 0);
      }
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
  HMOE_REQUIRE_CODE(d_model >= 128 && d_model % 128 == 0 && d_model <= kMaxRowCols, HMOE_ERR_UNSUPPORTED,
                    "%s: d_model must be a multiple of 128 up to %d (got %d)", what, kMaxRowCols, d_model);
  HMOE_REQUIRE_CODE(d_ff >= 128 && d_ff % 128 == 0 && d_ff <= kMaxRowCols, HMOE_ERR_UNSUPPORTED,
                    "%s: d_ff must be a multiple of 128 up to %d (got %d)", what, kMaxRowCols, d_ff);
  return HMOE_OK;
}

// What a launch cannot count in 32 bits beyond that: the tiles of the smaller tile form.
// (An expert's columns of a tile are 256 x 32768 bytes, its rows 128 x 65536 x 2.)
bool too_many_tiles(int64_t rows_cap, int n_experts, int ncols) {
  return (ceil_div(rows_cap, 64) + n_experts) * ceil_div(ncols, kTileN) > (int64_t(1) << 30);
}

// Which kernel a product takes: the one with the least estimated time, from measured
// rates (MI355X, us, `steps` = K / 128):
//   rows: 3.3, and 1.15 ns for every 32 rows x 64 columns x 128 values, or 0.72 a step (split
//     over four waves 0.19); or the experts' weights at 5.0 TB/s and, for every 64 columns, the
//     rows at 27;
//   64-row tiles, three a CU at a time: 4.0, and for each that a CU has 0.36 a step (0.465 for one
//     alone) and 0.42; or the weights and 1.5;
//   128-row tiles, two a CU: 4.2, 0.545 (0.632) and 1.65; or the weights and 1.5.
// Measured against each other (rows, rows split, 64, 128), us:
//   gate/up 64 experts, D 2048, F 1024, top-8: 1 token 13.4, 7.4, 12.3, 17.2; 48 tokens 41.8,
//     41.5, 45.4, 44.3; 256 tokens 61, 52, 53.5, 45.7; 384 tokens 67, 69, 49.6, 63; 1000 tokens
//     129, 139, 65, 60; 4000 tokens 407, 436, 194, 147; 16384 tokens 1496, 1610, 730, 500;
//   32 experts, D 4096, F 2048, top-4: 48 tokens 88, 100, 102, 90; 300 tokens 131, 131, 107, 121;
//   24 experts, D 1152, F 640, top-3: 100 tokens 14.2, 8.9, 10.7, 13.1; 333 tokens 15.6, 15.9,
//     11.5, 14.6; 1500 tokens 31, 32, 14.6, 16.4;
//   one segment, D 2048, F 1024: 200 rows 15.2, 6.8, 11.2, 16.9; 8000 rows 103, 113, 45, 39.
// Over 182 such products the rule's choice is 1 % slower than the fastest on average, 21 % at most.
enum Form { kRows1, kRows4, kTiles64, kTiles128 };

Form choose_form(int64_t rows, int n_experts, int kdim, int ncols, int cus) {
  const double steps = kdim / 128;
  const double weights = live_experts(rows, n_experts) * ncols * static_cast<double>(kdim) / 5.0e6;
  const double re_read = static_cast<double>(rows) * (ncols / 64) * kdim / 27e6;
  const double waves = row_tiles(rows, n_experts, 32) * (ncols / 64);
  const bool split = steps >= 2 && waves < 5.0 * cus;  // (more waves side by side fill the chip)
  const double by_rows =
      std::max({3.3 + waves * steps * 1.15e-3, 3.3 + steps * (split ? 0.19 : 0.72), weights + re_read + 1.0});
  const auto by_tiles = [&](int bm, int per_cu, double start, double alone, double busy, double end) {
    const double tiles = row_tiles(rows, n_experts, bm) * static_cast<double>(ceil_div(ncols, kTileN));
    const double whole = std::floor(tiles / (per_cu * cus)), rest = tiles - whole * per_cu * cus;
    const double last = rest < 1.0 ? 0.0 : std::max(1.0, std::ceil(rest / cus - 0.02));  // of a CU
    return std::max(start + steps * (whole * per_cu * busy + (last > 0.0 ? std::max(alone, busy * last) : 0.0)) +
                        end * (whole * per_cu + last),
                    weights + 1.5);
  };
  const double by_64 = by_tiles(64, TileCfg<64, true>::kPerCu, 4.0, 0.465, 0.36, 0.42);
  const double by_128 = by_tiles(128, TileCfg<128, true>::kPerCu, 4.2, 0.632, 0.545, 1.65);
  // (a grid holds 65535 tiles along y)
  if (by_rows <= std::min(by_64, by_128) && max_row_tiles(rows, n_experts) <= 65535)
    return split ? kRows4 : kRows1;
  return by_64 <= by_128 ? kTiles64 : kTiles128;
}

template <bool GATE_UP, bool GATHER>
int launch_product(const char* what, const int8_t* a, const float* a_scale, const int8_t* b, const float* b_scale,
                   const int32_t* offsets, int n_experts, int64_t rows_cap, int kdim, int ncols, void* c,
                   const int32_t* gather_src, int gather_k, int gather_rows, hipStream_t s) {
  const Divisor by_k = divisor(gather_k);
  HMOE_REQUIRE(!too_many_tiles(rows_cap, n_experts, ncols), "%s: too many tiles", what);
  uint16_t* const out = static_cast<uint16_t*>(c);
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
      if (int rc = allow_lds(what, grouped_i8_tiles<bm, GATE_UP, GATHER>, lds, dev, &done)) return rc;
      hipLaunchKernelGGL((grouped_i8_tiles<bm, GATE_UP, GATHER>), dim3(per_cu * cus), dim3(kTileThreads), lds, s, a,
                         a_scale, b, b_scale, offsets, n_experts, kdim, ncols, out, gather_src, by_k, gather_rows,
                         by_cols, by_group);
      return check_launch(what);
    };
    return form == kTiles64 ? launch(std::integral_constant<int, 64>{}) : launch(std::integral_constant<int, 128>{});
  }
  const unsigned m_tiles = static_cast<unsigned>(max_row_tiles(rows_cap, n_experts));
  if (form == kRows4)
    hipLaunchKernelGGL((grouped_i8_rows<GATE_UP, GATHER, 4>), dim3(ncols / 64, m_tiles), dim3(256), 0, s, a, a_scale,
                       b, b_scale, offsets, n_experts, kdim, ncols, out, gather_src, by_k, gather_rows);
  else
    hipLaunchKernelGGL((grouped_i8_rows<GATE_UP, GATHER, 1>),
                       dim3(static_cast<unsigned>(ceil_div(ncols, 256)), m_tiles), dim3(256), 0, s, a, a_scale, b,
                       b_scale, offsets, n_experts, kdim, ncols, out, gather_src, by_k, gather_rows);
  return check_launch(what);
}

}  // namespace
}  // namespace hmoe

extern "C" int64_t hmoe_grouped_i8_form(int64_t rows_cap, int n_experts, int kdim, int ncols, int cus) {
  using namespace hmoe;
  if (rows_cap < 1 || rows_cap > kMaxRows || n_experts < 1 || n_experts > kMaxExperts || cus < 1 || kdim < 128 ||
      kdim % 128 != 0 || kdim > kMaxRowCols || ncols < 128 || ncols % 128 != 0 || ncols > 2 * kMaxRowCols ||
      too_many_tiles(rows_cap, n_experts, ncols)) {
    set_error("grouped_i8_form: sizes that the products refuse");
    return -1;
  }
  return choose_form(rows_cap, n_experts, kdim, ncols, cus);
}

extern "C" int hmoe_grouped_gate_up_i8(const int8_t* xs_q, const float* xs_scale, const int32_t* offsets,
                                       int n_experts, int64_t rows_cap, int d_model, int d_ff, const int8_t* w_packed,
                                       const float* w_scales, void* h, hmoe_stream_t stream) {
  using namespace hmoe;
  const char* what = "grouped_gate_up_i8";
  if (int rc = check_product(what, n_experts, rows_cap, d_model, d_ff)) return rc;
  if (rows_cap == 0) return HMOE_OK;
  HMOE_REQUIRE(xs_q && xs_scale && offsets && w_packed && w_scales && h, "%s: null pointer argument", what);
  HMOE_REQUIRE_ALIGNED(what, 16, xs_q, w_packed, w_scales, h);
  return launch_product<true, false>(what, xs_q, xs_scale, w_packed, w_scales, offsets, n_experts, rows_cap, d_model,
                                     2 * d_ff, h, nullptr, 1, 1, static_cast<hipStream_t>(stream));
}

extern "C" int hmoe_grouped_gate_up_i8_gather(const int8_t* x_q, const float* x_scale, int64_t tokens, int top_k,
                                              const int32_t* perm_src, const int32_t* offsets, int n_experts,
                                              int64_t rows_cap, int d_model, int d_ff, const int8_t* w_packed,
                                              const float* w_scales, void* h, hmoe_stream_t stream) {
  using namespace hmoe;
  const char* what = "grouped_gate_up_i8_gather";
  if (int rc = check_product(what, n_experts, rows_cap, d_model, d_ff)) return rc;
  HMOE_REQUIRE(tokens >= 0 && top_k >= 1 && (tokens >= 1 || rows_cap == 0),
               "%s: need tokens >= 0, top_k >= 1 (tokens >= 1 with rows)", what);
  HMOE_REQUIRE(tokens < (int64_t(1) << 31) && tokens * d_model < (int64_t(1) << 31),
               "%s: x_q must be smaller than 2 GiB", what);
  if (rows_cap == 0) return HMOE_OK;
  HMOE_REQUIRE(x_q && x_scale && perm_src && offsets && w_packed && w_scales && h, "%s: null pointer argument", what);
  HMOE_REQUIRE_ALIGNED(what, 16, x_q, w_packed, w_scales, h);
  return launch_product<true, true>(what, x_q, x_scale, w_packed, w_scales, offsets, n_experts, rows_cap, d_model,
                                    2 * d_ff, h, perm_src, top_k, static_cast<int>(tokens),
                                    static_cast<hipStream_t>(stream));
}

extern "C" int hmoe_grouped_down_i8(const int8_t* h_q, const float* h_scale, const int32_t* offsets, int n_experts,
                                    int64_t rows_cap, int d_ff, int d_model, const int8_t* w_packed,
                                    const float* w_scales, void* ys, hmoe_stream_t stream) {
  using namespace hmoe;
  const char* what = "grouped_down_i8";
  if (int rc = check_product(what, n_experts, rows_cap, d_model, d_ff)) return rc;
  if (rows_cap == 0) return HMOE_OK;
  HMOE_REQUIRE(h_q && h_scale && offsets && w_packed && w_scales && ys, "%s: null pointer argument", what);
  HMOE_REQUIRE_ALIGNED(what, 16, h_q, w_packed, w_scales, ys);
  return launch_product<false, false>(what, h_q, h_scale, w_packed, w_scales, offsets, n_experts, rows_cap, d_ff,
                                      d_model, ys, nullptr, 1, 1, static_cast<hipStream_t>(stream));
}
