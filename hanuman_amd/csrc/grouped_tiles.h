// What the grouped products on packed operands share (MXFP4 and int8): finding an
// expert's row tiles, the tiles' order, loads into LDS and their waits, storing bf16
// rows, and the counts that the choice of a kernel goes by.
#pragma once

#include <algorithm>
#include <atomic>
#include <cmath>

#include "hmoe_common.h"

namespace hmoe {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int64_t kMaxRows = int64_t(1) << 30;
constexpr int kMaxDim = 1 << 20;  // of D and F
constexpr int kBufferWord3 = 0x00020000;
constexpr int kNonTemporal = 2;  // cache policy of a buffer access

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pack_bf16x2_rne(float lo, float hi) {
  f32x2_t v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
}

// silu(g) u, off by at most (1.25 |g| + 8) 2^-24 of itself: the exponential's argument g
// log2(e) is rounded once, a quarter more is log2(e)'s own rounding, and the hardware's
// exponential and reciprocal are good to a float32 step, the sum and products to half a one.
// Below g = -87.3 (1 + e^-g past 2^126) the reciprocal is subnormal and may come out as
// zero: up to |g u| 2^-126 is lost there.  Sums past float32's range give infinity or NaN.
__device__ __forceinline__ float swiglu_f32(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.0f + __expf(-g)) * u;
}

// n / d for 0 <= n < 2^31 without a division: with 2^s the first power of two that is not
// below d, mul = ceil(2^(31 + s) / d) is too large by less than 2^s / d, which n times over
// is less than the 2^(31 + s) / d that the quotient could be off by.
struct Divisor {
  uint32_t mul;
  int shift;
};
Divisor divisor(int d) {
  int s = 0;
  while ((int64_t(1) << s) < d) ++s;
  return {static_cast<uint32_t>(((uint64_t(1) << (31 + s)) + d - 1) / d), s};
}
__device__ __forceinline__ int divide(int n, Divisor d) {
  return static_cast<int>(__umulhi(static_cast<uint32_t>(n) * 2u, d.mul) >> d.shift);
}

// The token of a row's slot; a row without a source reads token 0.
__device__ __forceinline__ int token_of(int32_t slot, Divisor top_k, int tokens) {
  const int t = divide(slot > 0 ? slot : 0, top_k);
  return t < tokens ? t : tokens - 1;
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

// Lane L of an accumulator holds row L % 32 of A's fragment and columns 8 q + 4 (L / 32)
// + 0..3 (q = 0..3) of B's.
//
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

// Memory accesses are not moved past it by the compiler.
__device__ __forceinline__ void order_memory() { asm volatile("" ::: "memory"); }

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
  order_memory();  // (a lane reads what others wrote; a wave's LDS accesses run in their order)
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const int rr = 8 * m + (lane >> 3);
    const u32x4 v = *reinterpret_cast<const u32x4*>(lds + rr * 128 + (((lane & 7) ^ (rr & 7)) * 16));
    __builtin_amdgcn_raw_buffer_store_b128(v, out, ((row0 + rr) * ldc + col + (lane & 7) * 8) * 2, 0, kNonTemporal);
  }
  order_memory();  // (the next blocks' writes stay behind these reads)
}

constexpr int kNumXcd = 8;
constexpr int kTileN = 256;
constexpr int kTileGroup = 8;

typedef __attribute__((address_space(3))) void* lds_ptr_t;

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint8_t* dst, uint32_t voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)dst, 16, voff, 0, 0, 0);
}

// A use that later code is not moved before.  (A function of its own, like dma16:
// where the operand's type depends on a template the host pass drops the kernel.)
__device__ __forceinline__ void use_here(const f32x16& v) { asm volatile("" ::"v"(v)); }

__device__ __forceinline__ int swz128(int r) { return (r >> 1) & 7; }

// order_memory, for instructions of every kind.
__device__ __forceinline__ void fence() {
  order_memory();
  __builtin_amdgcn_sched_barrier(0);
}

// s_waitcnt lgkmcnt(0)
__device__ __forceinline__ void wait_lgkm0() { __builtin_amdgcn_s_waitcnt(0xc07f); }

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
  // On to tile t (t grows from call to call; by_cols, by_group: the column tiles, a group's
  // tiles).
  __device__ __forceinline__ void move(const int32_t* __restrict__ offsets, int t, int n_tiles_n, Divisor by_cols,
                                       Divisor by_group) {
    const int m_any = divide(t, by_cols);
    while (m_any >= before + tiles) {
      before += tiles;
      expert(offsets, e + 1);
    }
    const int u = t - before * n_tiles_n;
    const int g = divide(u, by_group);
    const int left = tiles - g * kTileGroup;
    const int gm = left < kTileGroup ? left : kTileGroup;
    const int v = u - g * kTileGroup * n_tiles_n;
    const int n_tile = gm == kTileGroup ? v / kTileGroup : v / gm;
    row0 = seg0 + (g * kTileGroup + (v - n_tile * gm)) * BM;
    rows = seg1 - row0 < BM ? seg1 - row0 : BM;
    n0 = n_tile * kTileN;
  }
};

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

}  // namespace
}  // namespace hmoe
