// Top-k among the experts of the best groups.  The N experts are G groups of N / G; a group's
// score is its largest key (softmax; a key is a logit) or the float32 sum of its two largest
// (sigmoid; a key is the score plus the bias).  The top_groups groups with the largest scores
// keep their experts, the top_k of these with the largest keys are taken, in both the lower
// index first where equal (totalOrder).  A sum that is NaN is below every score, since the sign of
// an arithmetic's NaN says nothing; a logit that is NaN keeps its place in totalOrder, as without
// groups.  Gates as without groups.
//
// A token has 2^log_lanes lanes: groups g = 0 .. G padded to a power of two, 2^log_lg each, E keys in
// each lane's registers.  A key and its expert are one positive float64 that orders like the
// pair, so that a comparison-and-exchange is a maximum and a minimum.  Each lane sorts its keys
// into a list of the eight, sixteen or 32 largest (top_k and more; a sorting network over eights,
// merged), which also gives a group's two largest; lanes of groups that are not taken empty
// theirs, and the token's lists are merged over its lanes.
//
// Bound by vector instructions, 85 a key, of which the sigmoid is 26 (its single operations are
// what makes the choice the same everywhere) and the lists the rest: 16384 tokens on 256 experts
// 11.3 us (captured again and again; 12.3 traced from Python), of which the logits' 17 MB are
// 3.7.  In rounds, the largest of all taken each time, with keys compared as two integers, they
// took 30 us; with sigmoid_det's range checks and division 13.5.  Twelve experts a token 14 us (in rounds on these keys 21), 32 21 us (39); one token 4.8, 6.2
// and 9.1 us (9.9 and 18.7 in rounds).
#pragma once

#include <type_traits>

#include "hmoe_common.h"

namespace hmoe {

constexpr int kMaxGroups = 64;
constexpr int kList = 8, kLongList = 16, kLongestList = 32;

struct GroupRule {
  int n_experts, n_groups, top_groups, top_k, mode;
  float rsf;
  int size;        // experts of a group
  int log_lg;      // log2 of a group's lanes
  int log_lanes;   // log2 of a token's lanes, 3 and more
};

// Lanes for E keys each.
inline GroupRule group_rule(int n_experts, int n_groups, int top_groups, int top_k, int mode, float rsf, int keys) {
  GroupRule r{n_experts, n_groups, top_groups, top_k, mode, rsf, n_experts / n_groups, 0, 0};
  int log_groups = 0;
  while ((1 << log_groups) < n_groups) ++log_groups;
  while ((keys << r.log_lg) < r.size || log_groups + r.log_lg < 3) ++r.log_lg;
  r.log_lanes = log_groups + r.log_lg;
  return r;
}

// Words of LDS for `count` values and the run of 32 that may be read past them, four more for
// every 32.
__host__ __device__ inline int group_stage_words(int count) { return (count / 32 + 2) * 36; }

// sigmoid_det for |x| < 87, the same bits: the range checks cannot hold there, and the
// reciprocal of 1 + e^-x < 2^126 is correctly rounded after one step of Newton's iteration on
// the hardware's (looked at for every float32 from 1 to 2^126).
__device__ __forceinline__ float sigmoid_near(float x) {
#pragma clang fp contract(off)
  const float n = __builtin_rintf(-x * __uint_as_float(0x3fb8aa3bu));
  float r = -x - n * __uint_as_float(0x3f317200u);
  r = r - n * __uint_as_float(0x35bfbe8eu);
  float p = __uint_as_float(0x39500d01u);
  p = p * r + __uint_as_float(0x3ab60b61u);
  p = p * r + __uint_as_float(0x3c088889u);
  p = p * r + __uint_as_float(0x3d2aaaabu);
  p = p * r + __uint_as_float(0x3e2aaaabu);
  p = p * r + 0.5f;
  p = p * r + 1.0f;
  p = p * r + 1.0f;
  const float d = 1.0f + __builtin_ldexpf(p, static_cast<int>(n));
  const float y = __builtin_amdgcn_rcpf(d);
  return __builtin_fmaf(__builtin_fmaf(-d, y, 1.0f), y, y);
}

// (key, index) as a float64: totalOrder of the key, then the lower index, below 256.  Bit 61
// is set, so that it is neither a NaN nor subnormal and above kNone.
constexpr double kNone = 0.0;
__device__ __forceinline__ double ranked(float key, int index) {
  const uint32_t b = __float_as_uint(key);
  const uint32_t u = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
  const uint64_t w = (static_cast<uint64_t>(0x20000000u | (u >> 3)) << 32) | ((u << 29) | static_cast<uint32_t>(255 - index));
  return __builtin_bit_cast(double, w);
}
__device__ __forceinline__ int ranked_index(double v) {
  return 255 - static_cast<int>(__builtin_bit_cast(uint64_t, v) & 255u);
}
__device__ __forceinline__ float ranked_key(double v) {
  const uint32_t u = static_cast<uint32_t>(__builtin_bit_cast(uint64_t, v) >> 29);
  return __uint_as_float(u ^ ((u & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}

__device__ __forceinline__ double dmax(double a, double b) { return __builtin_fmax(a, b); }
__device__ __forceinline__ double dmin(double a, double b) { return __builtin_fmin(a, b); }
__device__ __forceinline__ void order2(double& a, double& b) {  // the larger one first
  const double hi = dmax(a, b);
  b = dmin(a, b);
  a = hi;
}

// v of the lane that the DPP control names.
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t w = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_mov_dpp(static_cast<int32_t>(w), CTRL, 0xF, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_mov_dpp(static_cast<int32_t>(w >> 32), CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}
// The values of both blocks of 16 (32) lanes, in the same order in both.
template <int WIDTH>
__device__ __forceinline__ void both_blocks(double v, double& first, double& second) {
  const uint64_t w = __builtin_bit_cast(uint64_t, v);
  const uint32_t l = static_cast<uint32_t>(w), h = static_cast<uint32_t>(w >> 32);
  const auto lo = WIDTH == 16 ? __builtin_amdgcn_permlane16_swap(l, l, false, false)
                              : __builtin_amdgcn_permlane32_swap(l, l, false, false);
  const auto hi = WIDTH == 16 ? __builtin_amdgcn_permlane16_swap(h, h, false, false)
                              : __builtin_amdgcn_permlane32_swap(h, h, false, false);
  first = __builtin_bit_cast(double, (static_cast<uint64_t>(hi[0]) << 32) | lo[0]);
  second = __builtin_bit_cast(double, (static_cast<uint64_t>(hi[1]) << 32) | lo[1]);
}
// Of lanes that agree in blocks of 2^LOG: the value of this lane's block and of the block
// beside it (in an order of its own in each pair of blocks).
template <int LOG>
__device__ __forceinline__ void beside(double v, double& a, double& b) {
  constexpr int kCtrl = LOG == 0 ? 0xB1 : LOG == 1 ? 0x4E : LOG == 2 ? 0x141 : 0x140;
  if constexpr (LOG >= 4) {
    both_blocks<LOG == 4 ? 16 : 32>(v, a, b);
  } else {
    a = v;
    b = dpp_f64<kCtrl>(v);
  }
}

// f(LOG) for LOG from lo on below hi (uniform), in order.
template <typename F>
__device__ __forceinline__ void for_logs(int lo, int hi, F f) {
  if (lo <= 0 && hi > 0) f(std::integral_constant<int, 0>{});
  if (lo <= 1 && hi > 1) f(std::integral_constant<int, 1>{});
  if (lo <= 2 && hi > 2) f(std::integral_constant<int, 2>{});
  if (lo <= 3 && hi > 3) f(std::integral_constant<int, 3>{});
  if (lo <= 4 && hi > 4) f(std::integral_constant<int, 4>{});
  if (lo <= 5 && hi > 5) f(std::integral_constant<int, 5>{});
}

// Eight values in descending order, with 19 exchanges.
__device__ __forceinline__ void sort8(double (&c)[8]) {
  constexpr int kPairs[19][2] = {{0, 1}, {2, 3}, {4, 5}, {6, 7}, {0, 2}, {1, 3}, {4, 6}, {5, 7}, {1, 2}, {5, 6},
                                 {0, 4}, {3, 7}, {1, 5}, {2, 6}, {1, 4}, {3, 6}, {2, 4}, {3, 5}, {3, 4}};
#pragma unroll
  for (int i = 0; i < 19; ++i) order2(c[kPairs[i][0]], c[kPairs[i][1]]);
}
// Values that rise and then fall, or the other way, in descending order.
template <int L>
__device__ __forceinline__ void order_bitonic(double (&a)[L]) {
#pragma unroll
  for (int d = L / 2; d > 0; d /= 2)
#pragma unroll
    for (int i = 0; i < L; ++i)
      if ((i & d) == 0) order2(a[i], a[i + d]);
}
// a: the L largest of a and b, both descending.
template <int L>
__device__ __forceinline__ void merge_lists(double (&a)[L], const double (&b)[L]) {
#pragma unroll
  for (int i = 0; i < L; ++i) a[i] = dmax(a[i], b[L - 1 - i]);
  order_bitonic(a);
}
// list: the L largest of c, descending.
template <int E, int L>
__device__ __forceinline__ void sort_list(const double (&c)[E], double (&list)[L]) {
  static_assert(E == 8 || E == 16, "keys of a lane");
  double part[E];
#pragma unroll
  for (int i = 0; i < E; ++i) part[i] = c[i];
  if constexpr (E == 8) {
    sort8(part);
  } else {
    double a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = c[i];
      b[i] = c[8 + i];
    }
    sort8(a);
    sort8(b);
    if constexpr (L == 8) merge_lists(a, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      part[i] = a[i];
      part[15 - i] = b[i];
    }
    if constexpr (L > 8) order_bitonic(part);
  }
#pragma unroll
  for (int i = 0; i < L; ++i) list[i] = i < E ? part[i < E ? i : 0] : kNone;
}

// How many of the token's lanes hold a larger value than this one.
__device__ __forceinline__ int count_above8(double mine, double v) {
  const double m = dpp_f64<0x141>(v);  // lane 7 - i of eight
  return (v > mine) + (dpp_f64<0xB1>(v) > mine) + (dpp_f64<0x4E>(v) > mine) + (dpp_f64<0x1B>(v) > mine) + (m > mine) +
         (dpp_f64<0xB1>(m) > mine) + (dpp_f64<0x4E>(m) > mine) + (dpp_f64<0x1B>(m) > mine);
}
__device__ __forceinline__ int count_above16(double mine, double v, int log_lanes) {
  int n = count_above8(mine, v);
  if (log_lanes > 3) n += count_above8(mine, dpp_f64<0x140>(v));  // lane 15 - i of sixteen
  return n;
}
__device__ __forceinline__ int count_above(double v, int log_lanes) {
  if (log_lanes <= 4) return count_above16(v, v, log_lanes);
  double a, b;
  both_blocks<16>(v, a, b);
  int n = 0;
  if (log_lanes == 5) return count_above16(v, a, 4) + count_above16(v, b, 4);
  double a0, a1, b0, b1;
  both_blocks<32>(a, a0, a1);
  both_blocks<32>(b, b0, b1);
  n += count_above16(v, a0, 4) + count_above16(v, a1, 4);
  n += count_above16(v, b0, 4) + count_above16(v, b1, 4);
  return n;
}

// Selection and gates of one token by its lanes.  run(e, l, b): the logits and (sigmoid) the
// biases of E experts from e on, anything past the last one; get(e): the logit of one.  Every
// lane of the wave takes part; `store` says whether the token is there.  L: the lists' length,
// top_k and more.
template <int E, int L, typename Run, typename Get>
__device__ __forceinline__ void select_in_groups(Run run, Get get, const GroupRule& r, bool store,
                                                 int32_t* __restrict__ idx_row, float* __restrict__ gates_row) {
#pragma clang fp contract(off)
  const int lane = threadIdx.x & 63;
  const int lanes = 1 << r.log_lanes;
  const int p = lane & (lanes - 1);  // of the token's lanes
  const int group = p >> r.log_lg;
  const int in0 = (p & ((1 << r.log_lg) - 1)) * E;  // of the group
  const int e0 = group * r.size + in0;
  const int live = group < r.n_groups ? r.size - in0 : 0;  // of this lane's keys
  const bool sigmoid = r.mode == HMOE_ROUTE_SIGMOID_BIAS;
  double c[E];
  float l[E], b[E];
  run(live > 0 ? e0 : 0, l, b);
  if (sigmoid) {
    bool near = true;
#pragma unroll
    for (int j = 0; j < E; ++j) near = near && (j >= live || __builtin_fabsf(l[j]) < 87.0f);
    if (near) {
#pragma unroll
      for (int j = 0; j < E; ++j) l[j] = sigmoid_near(l[j]) + b[j];
    } else {
#pragma unroll 1
      for (int j = 0; j < E; ++j) l[j] = sigmoid_det(l[j]) + b[j];
    }
  }
#pragma unroll
  for (int j = 0; j < E; ++j) c[j] = j < live ? ranked(l[j], e0 + j) : kNone;

  double list[L];
  sort_list(c, list);
  // the group's two largest
  double best1 = list[0], best2 = list[1];
  for_logs(0, r.log_lg, [&](auto log) __attribute__((always_inline)) {
    double a1, b1, a2, b2;
    beside<decltype(log)::value>(best1, a1, b1);
    beside<decltype(log)::value>(best2, a2, b2);
    best1 = dmax(a1, b1);
    best2 = dmax(dmin(a1, b1), dmax(a2, b2));
  });
  double score = kNone;
  if (group < r.n_groups) {
    float s = ranked_key(best1);
    if (sigmoid) s = s + ranked_key(best2);
    score = ranked(sigmoid && s != s ? __uint_as_float(0xffffffffu) : s, group);
  }
  // (a group's lanes hold the same score)
  const bool taken = count_above(score, r.log_lanes) < r.top_groups << r.log_lg;

#pragma unroll
  for (int i = 0; i < L; ++i) list[i] = taken ? list[i] : kNone;
  for_logs(0, r.log_lanes, [&](auto log) __attribute__((always_inline)) {
    double other[L];
#pragma unroll
    for (int i = 0; i < L; ++i) {
      double a, b;
      beside<decltype(log)::value>(list[i], a, b);
      list[i] = a;
      other[i] = b;
    }
    merge_lists(list, other);
  });
  // slot k of the token is kept by lane k % lanes, as its (k / lanes)th (a token has eight lanes
  // at least)
  constexpr int kSlots = L / 8;
  double mine[kSlots];
#pragma unroll
  for (int q = 0; q < kSlots; ++q) {
    mine[q] = kNone;
#pragma unroll
    for (int i = 8 * q; i < L; ++i) mine[q] = p == i - (q << r.log_lanes) ? list[i] : mine[q];
  }
  // gates, summed in the slots' order
  int at[kSlots];
  float value[kSlots];
#pragma unroll
  for (int q = 0; q < kSlots; ++q) {
    // (a slot past top_k may hold nothing)
    at[q] = (q << r.log_lanes) + p < r.top_k ? ranked_index(mine[q]) : 0;
    value[q] = get(at[q]);
    if (sigmoid) value[q] = sigmoid_det(value[q]);
  }
  const int first = lane - p;
  if (!sigmoid) {
    const float most = __shfl(value[0], first);
#pragma unroll
    for (int q = 0; q < kSlots; ++q) value[q] = exp_det(value[q] - most);
  }
  float v[L];
#pragma unroll
  for (int k = 0; k < L; ++k) {
    float of = value[0];
#pragma unroll
    for (int q = 1; q <= k / 8; ++q) of = k >> r.log_lanes == q ? value[q] : of;
    v[k] = __shfl(of, first + (k & (lanes - 1)));
  }
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < L; ++k) sum = k < r.top_k ? sum + v[k] : sum;
#pragma unroll
  for (int q = 0; q < kSlots; ++q) {
    const int k = (q << r.log_lanes) + p;
    if (store && k < r.top_k) {
      idx_row[k] = at[q];
      gates_row[k] = sigmoid ? (value[q] / (sum + 1e-9f)) * r.rsf : value[q] / sum;
    }
  }
}

}  // namespace hmoe
