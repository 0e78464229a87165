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
#include <atomic>
#include <type_traits>

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

// ---- tiles for experts with many rows ------------------------------------------
// One workgroup of eight waves a CU loops over BM x 256 tiles.  A K step is 128
// values = 64 bytes of every row; the operands go from global memory into a ring of
// four LDS stages (buffer_load ... lds), three steps ahead and on into the next
// tile.  A's part of a stage has 64-byte rows whose 16-byte chunk c sits at c ^
// swz64(r), so that 16 lanes of a fragment read cover all banks; B's is the
// operand's own blocks of 1 KB, read lane by lane.  A step is two sub-steps of one
// MFMA per pair of fragments; the fragments of the next sub-step are read during
// each, so one barrier a step suffices: it is passed with the step after next in
// LDS.  The exponents of four steps come together (16 bytes of every row of A, 1 KB
// of B a step) into one of three regions, by one instruction of each wave.  (A tile's
// last group may be one step: the steps being loaded then span three groups.)
constexpr int kTileThreads = 512;
constexpr int kStages = 4;
constexpr int kRegions = 3;
constexpr int kNumXcd = 8;
constexpr int kTileN = 256;
constexpr int kTileGroup = 8;

template <int BM>
struct TileCfg {
  static constexpr int kA = BM * 64, kB = kTileN * 64;
  static constexpr int kStage = kA + kB;
  static constexpr int kExA = BM * 16, kExB = kTileN * 16;
  static constexpr int kEx = kExA + kExB;
  static constexpr int kLds = kStages * kStage + kRegions * kEx;
  static constexpr int kNA = BM / 128, kNB = kTileN / 128;  // DMA instructions a wave and step
  static constexpr int kFR = BM / 64;                       // row fragments a wave
};

typedef __attribute__((address_space(3))) void* lds_ptr_t;

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint8_t* dst, uint32_t voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)dst, 16, voff, soff, 0, 0);
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

// Exclusive scan of the experts' counts of BM-row tiles into tstart[0 .. n_experts].
template <int BM>
__device__ __forceinline__ int scan_tiles(const int32_t* __restrict__ offsets, int n_experts, int32_t* tstart,
                                          int32_t* tmp) {
  constexpr int kPer = kMaxExperts / kTileThreads;
  const int tid = threadIdx.x;
  int local[kPer], sum = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = tid * kPer + j;
    local[j] = e < n_experts ? (offsets[e + 1] - offsets[e] + BM - 1) / BM : 0;
    sum += local[j];
  }
  tmp[tid] = sum;
  __syncthreads();
  for (int off = 1; off < kTileThreads; off <<= 1) {
    const int v = tid >= off ? tmp[tid - off] : 0;
    __syncthreads();
    tmp[tid] += v;
    __syncthreads();
  }
  int run = tmp[tid] - sum;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = tid * kPer + j;
    if (e < n_experts) tstart[e] = run;
    run += local[j];
  }
  if (tid == kTileThreads - 1) tstart[n_experts] = tmp[kTileThreads - 1];
  __syncthreads();
  return tstart[n_experts];
}

struct Tile {
  int e, row0, rows, n0;
};

template <int BM, bool GATE_UP, bool GATHER>
__global__ __launch_bounds__(kTileThreads) void grouped_mxfp4_tiles(
    const uint8_t* __restrict__ A, const uint8_t* __restrict__ a_exp, const uint8_t* __restrict__ B,
    const uint8_t* __restrict__ b_exp, const int32_t* __restrict__ offsets, int n_experts, int kdim, int ncols,
    uint8_t* __restrict__ C, uint8_t* __restrict__ c_exp, const int32_t* __restrict__ gather_src, int gather_k,
    int gather_rows) {
  typedef TileCfg<BM> Cfg;
  constexpr int kNA = Cfg::kNA, kNB = Cfg::kNB, kFR = Cfg::kFR;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  __shared__ int32_t tstart[kMaxExperts + 1];
  __shared__ int32_t scan_tmp[kTileThreads];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n_tiles_n = ncols / kTileN;
  const int total = __builtin_amdgcn_readfirstlane(scan_tiles<BM>(offsets, n_experts, tstart, scan_tmp)) * n_tiles_n;
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

  // An expert's tiles in groups of kTileGroup row tiles, each swept column by
  // column (row tile fastest): an XCD's workgroups share few blocks of A and B.
  auto decode = [&](int t) __attribute__((always_inline)) {
    const int m_any = t / n_tiles_n;
    int l = 0, h = n_experts;  // largest e with tstart[e] <= m_any (it has a tile)
    while (h - l > 1) {
      const int mid = (l + h) >> 1;
      if (tstart[mid] <= m_any) l = mid; else h = mid;
    }
    const int e = __builtin_amdgcn_readfirstlane(l);
    const int ts = __builtin_amdgcn_readfirstlane(tstart[e]);
    const int me = __builtin_amdgcn_readfirstlane(tstart[e + 1]) - ts;
    const int u = t - ts * n_tiles_n;
    const int g = u / (kTileGroup * n_tiles_n);
    const int gm = me - g * kTileGroup < kTileGroup ? me - g * kTileGroup : kTileGroup;
    const int v = u - g * kTileGroup * n_tiles_n;
    const int n_tile = v / gm;
    Tile r;
    r.e = e;
    r.row0 = __builtin_amdgcn_readfirstlane(offsets[e]) + (g * kTileGroup + (v - n_tile * gm)) * BM;
    r.rows = __builtin_amdgcn_readfirstlane(offsets[e + 1]) - r.row0;
    r.rows = r.rows < BM ? r.rows : BM;
    r.n0 = n_tile * kTileN;
    return r;
  };

  // ---- load side -----------------------------------------------------------------
  // A: instruction j of wave w fills rows 16 (w kNA + j) + lane / 4, chunk (lane & 3)
  // ^ swz64(row).  B: blocks of 1 KB, block b = 2 (column / 32) + (64 values of the
  // step), instruction j of wave w block w kNB + j.
  const int a_row = 16 * wave * kNA + (lane >> 2);
  const int a_byte = ((lane & 3) ^ ((lane >> 4) & 3)) * 16;
  __amdgpu_buffer_rsrc_t a_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(A), 0,
                                                                    GATHER ? gather_rows * row_bytes : 0, kBufferWord3);
  __amdgpu_buffer_rsrc_t ae_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a_exp), 0,
                                                                     GATHER ? gather_rows * ex_bytes : 0, kBufferWord3);
  __amdgpu_buffer_rsrc_t b_rsrc = a_rsrc, be_rsrc = a_rsrc;
  uint32_t a_voff[kNA], ae_voff = 0, b_voff[kNB];
#pragma unroll
  for (int j = 0; j < kNB; ++j) {
    const int blk = wave * kNB + j;
    b_voff[j] = static_cast<uint32_t>((blk >> 1) * (kdim / 64) * 1024 + (blk & 1) * 1024 + lane * 16);
  }
  // waves 0 .. BM / 64 - 1 bring A's exponents, the next four B's (a step each)
  constexpr int kExWavesA = BM / 64;
  const bool ex_a = wave < kExWavesA, ex_b = wave >= kExWavesA && wave < kExWavesA + 4;
  int ld_kb = 0, ld_g = 0, ld_t = first, ld_region = 0;
  int32_t pf_src[kNA], pf_ex = 0;  // GATHER: sources of this lane's rows in the next tile
  auto fetch_src = [&](int t) __attribute__((always_inline)) {
    const Tile q = decode(t);
#pragma unroll
    for (int j = 0; j < kNA; ++j) {
      const int r = a_row + 16 * j;
      pf_src[j] = gather_src[q.row0 + (r < q.rows ? r : q.rows - 1)];
    }
    const int r = 64 * wave + lane;
    if (ex_a) pf_ex = gather_src[q.row0 + (r < q.rows ? r : q.rows - 1)];
  };
  auto token = [&](int32_t slot) __attribute__((always_inline)) {
    const int tk = slot >= 0 ? slot / gather_k : 0;  // a row without a source reads token 0
    return static_cast<uint32_t>(tk < gather_rows ? tk : gather_rows - 1);
  };
  auto set_load_tile = [&](int t) __attribute__((always_inline)) {
    const Tile q = decode(t);
    const int64_t block = static_cast<int64_t>(q.e) * (ncols / 32) + q.n0 / 32;
    b_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(B + block * (kdim / 64) * 1024), 0,
                                               kTileN * row_bytes, kBufferWord3);
    be_rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(b_exp + (static_cast<int64_t>(q.e) * ks * ncols + q.n0) * 4), 0,
        ((ks - 1) * ncols + kTileN) * 4, kBufferWord3);
    if (GATHER) {
#pragma unroll
      for (int j = 0; j < kNA; ++j) a_voff[j] = token(pf_src[j]) * static_cast<uint32_t>(row_bytes) + a_byte;
      ae_voff = token(pf_ex) * static_cast<uint32_t>(ex_bytes);
      if (t + per_xcd < hi) fetch_src(t + per_xcd);
    } else {
      // rows past the segment repeat its last one; their results are not stored
      a_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(A + static_cast<int64_t>(q.row0) * row_bytes), 0,
                                                 q.rows * row_bytes, kBufferWord3);
      ae_rsrc = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint8_t*>(a_exp + static_cast<int64_t>(q.row0) * ex_bytes), 0, q.rows * ex_bytes, kBufferWord3);
#pragma unroll
      for (int j = 0; j < kNA; ++j) {
        const int r = a_row + 16 * j;
        a_voff[j] = static_cast<uint32_t>((r < q.rows ? r : q.rows - 1) * row_bytes + a_byte);
      }
      const int r = 64 * wave + lane;
      ae_voff = static_cast<uint32_t>((r < q.rows ? r : q.rows - 1) * ex_bytes);
    }
  };
  // The exponents of steps ld_kb .. ld_kb + 3 (what a short last group reads past a
  // row's end is not used; past the buffer it is not read).
  auto issue_ex = [&]() __attribute__((always_inline)) {
    uint8_t* ex = smem + kStages * Cfg::kStage + ld_region * Cfg::kEx;
    if (ex_a) dma16(ae_rsrc, ex + wave * 1024, ae_voff + static_cast<uint32_t>(ld_kb * 4), 0);
    if (ex_b) {
      const int step = wave - kExWavesA;
      if (ld_kb + step < ks)
        dma16(be_rsrc, ex + Cfg::kExA + step * 1024, static_cast<uint32_t>(lane * 16), (ld_kb + step) * ncols * 4);
    }
  };
  auto issue_a = [&](int stage, int j) __attribute__((always_inline)) {
    dma16(a_rsrc, smem + stage * Cfg::kStage + (wave * kNA + j) * 1024, a_voff[j], ld_kb * 64);
  };
  auto issue_b = [&](int stage, int j) __attribute__((always_inline)) {
    dma16(b_rsrc, smem + stage * Cfg::kStage + Cfg::kA + (wave * kNB + j) * 1024, b_voff[j], ld_kb * 2048);
  };
  // (every step loaded: the last one again, into a stage that nothing reads, so
  // that a step always issues as many)
  bool ld_more = true;
  auto advance = [&]() __attribute__((always_inline)) {
    if (ld_g + 1 < iters) {
      ++ld_g;
      if (++ld_kb == ks) {
        ld_kb = 0;
        ld_t += per_xcd;
        set_load_tile(ld_t);
      }
      if ((ld_kb & 3) == 0) ld_region = ld_region + 1 == kRegions ? 0 : ld_region + 1;
    } else {
      ld_more = false;
    }
  };

  // ---- compute side ----------------------------------------------------------------
  // Wave w: rows (BM / 2) (w & 1) .. and columns 64 (w >> 1) .. of the tile.
  const int wm = wave & 1, wn = wave >> 1;
  const int frow = lane & 31, half = lane >> 5;
  const int fsw = swz64(frow);
  const int a_off = (wm * (BM / 2) + frow) * 64;
  const int b_off = Cfg::kA + wn * 4096 + lane * 16;
  u32x4 fa[2][kFR], fb[2][2];
  int exa[2][kFR], exb[2][2];
  auto read_frags = [&](auto Qc, int stage) __attribute__((always_inline)) {
    constexpr int q = decltype(Qc)::value;
    const uint8_t* st = smem + stage * Cfg::kStage;
#pragma unroll
    for (int j = 0; j < 2; ++j) fb[q][j] = *reinterpret_cast<const u32x4*>(st + b_off + j * 2048 + q * 1024);
#pragma unroll
    for (int i = 0; i < kFR; ++i)
      fa[q][i] = *reinterpret_cast<const u32x4*>(st + a_off + i * 2048 + (((2 * q + half) ^ fsw) * 16));
  };
  // Exponent words of a step, shifted so that byte 0 (2) is this lane's block of the
  // first (second) sub-step.
  auto read_ex = [&](auto Bc, int region, int kb) __attribute__((always_inline)) {
    constexpr int b = decltype(Bc)::value;
    const uint8_t* ex = smem + kStages * Cfg::kStage + region * Cfg::kEx;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      exb[b][j] = static_cast<int>(*reinterpret_cast<const uint32_t*>(
                                       ex + Cfg::kExA + (kb & 3) * 1024 + (wn * 64 + j * 32 + frow) * 4) >>
                                   (8 * half));
#pragma unroll
    for (int i = 0; i < kFR; ++i)
      exa[b][i] = static_cast<int>(*reinterpret_cast<const uint32_t*>(
                                       ex + (wm * (BM / 2) + i * 32 + frow) * 16 + (kb & 3) * 4) >>
                                   (8 * half));
  };
  f32x16 acc[kFR][2];

  int rd_kb = 0, rd_region = 0;  // the step whose fragments are read next
  auto rd_advance = [&]() __attribute__((always_inline)) {
    if (++rd_kb == ks) rd_kb = 0;
    if ((rd_kb & 3) == 0) rd_region = rd_region + 1 == kRegions ? 0 : rd_region + 1;
  };

  // Step g on exponent words b = g & 1.
  auto step = [&](auto Bc, int g) __attribute__((always_inline)) {
    constexpr int b = decltype(Bc)::value;
    const int stage = g & 3, next = (g + 1) & 3, fill = (g + 3) & 3;
    if (ld_more && (ld_kb & 3) == 0) issue_ex();
#pragma unroll
    for (int j = 0; j < kNA; ++j) issue_a(fill, j);
#pragma unroll
    for (int j = 0; j < kNB; ++j) issue_b(fill, j);
    advance();
    read_frags(std::integral_constant<int, 1>{}, stage);
#pragma unroll
    for (int i = 0; i < kFR; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = mfma_fp4<0>(fb[0][j], fa[0][i], acc[i][j], exb[b][j], exa[b][i]);
    read_frags(std::integral_constant<int, 0>{}, next);
    read_ex(std::integral_constant<int, b ^ 1>{}, rd_region, rd_kb);
    rd_advance();
#pragma unroll
    for (int i = 0; i < kFR; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = mfma_fp4<2>(fb[1][j], fa[1][i], acc[i][j], exb[b][j], exa[b][i]);
    // used here, before the barrier, so that the products are not moved past it
#pragma unroll
    for (int i = 0; i < kFR; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) use_here(acc[i][j]);
    // this wave's loads of step g + 2 have landed (step g + 3's may fly); after the
    // barrier every wave's have
    wait_vm_lgkm0<kNA + kNB>();
    __builtin_amdgcn_s_barrier();
  };

  if (GATHER) fetch_src(first);
  set_load_tile(first);
#pragma unroll
  for (int st = 0; st < 3; ++st) {
    if (ld_more && (ld_kb & 3) == 0) issue_ex();
#pragma unroll
    for (int j = 0; j < kNA; ++j) issue_a(st, j);
#pragma unroll
    for (int j = 0; j < kNB; ++j) issue_b(st, j);
    advance();
  }
  wait_vm_lgkm0<kNA + kNB>();
  __builtin_amdgcn_s_barrier();
  read_frags(std::integral_constant<int, 0>{}, 0);
  read_ex(std::integral_constant<int, 0>{}, 0, 0);
  rd_advance();

  int g = 0;
  for (int t = first; t < hi; t += per_xcd) {
#pragma unroll
    for (int i = 0; i < kFR; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    for (int kb = 0; kb < ks; ++kb, ++g) {
      step(std::integral_constant<int, 0>{}, g);
#pragma unroll
      for (int j = 0; j < 2; ++j) exb[0][j] = exb[1][j];
#pragma unroll
      for (int i = 0; i < kFR; ++i) exa[0][i] = exa[1][i];
    }
    const Tile q = decode(t);
    const int64_t r0 = q.row0;
    const int row = wm * (BM / 2) + frow;
    if constexpr (GATE_UP) {
      const int d_ff = ncols / 2;
      const __amdgpu_buffer_rsrc_t q_out =
          __builtin_amdgcn_make_buffer_rsrc(C + r0 * (d_ff / 2), 0, q.rows * (d_ff / 2), kBufferWord3);
      const __amdgpu_buffer_rsrc_t e_out =
          __builtin_amdgcn_make_buffer_rsrc(c_exp + r0 * (d_ff / 32), 0, q.rows * (d_ff / 32), kBufferWord3);
#pragma unroll
      for (int i = 0; i < kFR; ++i)
        store_h_block(acc[i][0], acc[i][1], q_out, e_out, row + 32 * i, q.n0 / 2 + wn * 32, d_ff, half);
    } else {
      const __amdgpu_buffer_rsrc_t out =
          __builtin_amdgcn_make_buffer_rsrc(C + r0 * ncols * 2, 0, q.rows * ncols * 2, kBufferWord3);
#pragma unroll
      for (int i = 0; i < kFR; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) store_y_block(acc[i][j], out, row + 32 * i, q.n0 + wn * 64 + 32 * j, ncols, half);
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

template <int BM, bool GATE_UP, bool GATHER, typename... Args>
int launch_tiles(const char* what, hipStream_t s, Args... args) {
  int dev = 0, grid = 0;
  if (int rc = persistent_grid(what, s, &grid, &dev)) return rc;
  static std::atomic<uint64_t> done{0};
  if (int rc = allow_lds(what, grouped_mxfp4_tiles<BM, GATE_UP, GATHER>, TileCfg<BM>::kLds, dev, &done)) return rc;
  hipLaunchKernelGGL((grouped_mxfp4_tiles<BM, GATE_UP, GATHER>), dim3(grid), dim3(kTileThreads), TileCfg<BM>::kLds, s,
                     args...);
  return check_launch(what);
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
  const double mean = static_cast<double>(rows_cap) / n_experts;
  if (mean >= 64 && ncols % kTileN == 0) {
    HMOE_REQUIRE(static_cast<int64_t>(kdim / 128) * ncols * 4 < (int64_t(1) << 31), "%s: operand too large", what);
    HMOE_REQUIRE((ceil_div(rows_cap, 128) + n_experts) * (ncols / kTileN) < (int64_t(1) << 31), "%s: too many tiles", what);
    if (mean >= 160)
      return launch_tiles<256, GATE_UP, GATHER>(what, s, a, a_exp, b, b_exp, offsets, n_experts, kdim, ncols, c, c_exp,
                                                gather_src, gather_k, gather_rows);
    return launch_tiles<128, GATE_UP, GATHER>(what, s, a, a_exp, b, b_exp, offsets, n_experts, kdim, ncols, c, c_exp,
                                              gather_src, gather_k, gather_rows);
  }
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
