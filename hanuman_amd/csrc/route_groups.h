// Top-k among the experts of the best groups.  The N experts are G groups of N / G; a group's
// score is its largest key (softmax; a key is a logit) or the float32 sum of its two largest
// (sigmoid; a key is the score plus the bias).  The top_groups groups with the largest scores
// keep their experts, the top_k of these with the largest keys are taken, in both the lower
// index first where equal (totalOrder).  A score that is NaN is below every other.  Gates as
// without groups.
//
// A token has L lanes: groups g = 0 .. G padded to a power of two, LG lanes for each, E keys in
// each lane's registers (one after another, so lanes are in the experts' order).  Scores are
// joined over a group's lanes, and a group's place is the number of groups ahead of it.  A
// round of the selection is two butterflies over the token's lanes, of the largest key and of
// the lowest expert that holds it.  Bound by the compares: a key costs a round four and a half
// instructions of the lane that holds it.
#pragma once

#include "hmoe_common.h"

namespace hmoe {

constexpr int kMaxGroups = 64;
constexpr int32_t kGone = INT32_MIN;  // below every key that is live

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

// v of the lane whose number differs in bit `log` alone.
__device__ __forceinline__ int32_t lane_xor(int32_t v, int log) {
  return __shfl_xor(v, 1 << log);
}

__device__ __forceinline__ int32_t imax(int32_t a, int32_t b) { return a > b ? a : b; }
__device__ __forceinline__ int32_t imin(int32_t a, int32_t b) { return a < b ? a : b; }

// The inverse of total_order_key.
__device__ __forceinline__ float key_value(int32_t k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }

// Selection and gates of one token by its lanes.  get(e): the logit of the token's expert e.
// Every lane of the wave takes part; `store` says whether the token is there.
template <int E, typename Get>
__device__ __forceinline__ void select_in_groups(Get get, const float* __restrict__ bias, const GroupRule& r,
                                                 bool store, int32_t* __restrict__ idx_row,
                                                 float* __restrict__ gates_row) {
#pragma clang fp contract(off)
  const int lane = threadIdx.x & 63;
  const int p = lane & ((1 << r.log_lanes) - 1);  // of the token's lanes
  const int first = lane - p;
  const int group = p >> r.log_lg;
  const int in0 = (p & ((1 << r.log_lg) - 1)) * E;  // of the group
  const int e0 = group * r.size + in0;
  const bool sigmoid = r.mode == HMOE_ROUTE_SIGMOID_BIAS;
  int32_t key[E];
  int32_t best1 = kGone, best2 = kGone;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const bool live = group < r.n_groups && in0 + j < r.size;
    float k = get(live ? e0 + j : 0);
    if (sigmoid) {
      k = sigmoid_det(k);
      if (bias != nullptr) k = k + bias[live ? e0 + j : 0];
    }
    key[j] = live ? imax(total_order_key(k), kGone + 1) : kGone;
    best2 = imax(best2, imin(best1, key[j]));
    best1 = imax(best1, key[j]);
  }
  for (int s = 0; s < r.log_lg; ++s) {
    const int32_t o1 = lane_xor(best1, s), o2 = lane_xor(best2, s);
    best2 = imax(imin(best1, o1), imax(best2, o2));
    best1 = imax(best1, o1);
  }
  int32_t score = best1;
  if (sigmoid) {
    const float sum = key_value(best1) + key_value(best2);
    score = sum != sum ? kGone + 1 : imax(total_order_key(sum), kGone + 1);
  }
  int ahead = 0;
  for (int g = 0; g < r.n_groups; ++g) {
    const int32_t other = __shfl(score, first + (g << r.log_lg));
    ahead += other > score || (other == score && g < group);
  }
  if (ahead >= r.top_groups) {
#pragma unroll
    for (int j = 0; j < E; ++j) key[j] = kGone;
  }
  int taken[4] = {0, 0, 0, 0};  // lane p has slots p, p + L, ... (a token has eight lanes at least)
  for (int k = 0; k < r.top_k; ++k) {
    int32_t most = key[0];
#pragma unroll
    for (int j = 1; j < E; ++j) most = imax(most, key[j]);
    for (int s = 0; s < r.log_lanes; ++s) most = imax(most, lane_xor(most, s));
    int32_t at = INT32_MAX;
#pragma unroll
    for (int j = E - 1; j >= 0; --j) at = key[j] == most ? e0 + j : at;
    for (int s = 0; s < r.log_lanes; ++s) at = imin(at, lane_xor(at, s));
#pragma unroll
    for (int j = 0; j < E; ++j) key[j] = at == e0 + j ? kGone : key[j];
    if ((k & ((1 << r.log_lanes) - 1)) == p) {
      const int slot = k >> r.log_lanes;
#pragma unroll
      for (int q = 0; q < 4; ++q) taken[q] = q == slot ? at : taken[q];
    }
  }
  // gates: slots in their order
  float value[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    value[q] = get(taken[q]);
    if (sigmoid) value[q] = sigmoid_det(value[q]);
  }
  if (!sigmoid) {
    const float most = __shfl(value[0], first);
#pragma unroll
    for (int q = 0; q < 4; ++q) value[q] = exp_det(value[q] - most);
  }
  float sum = 0.0f;
  for (int k = 0; k < r.top_k; ++k) {
    const int slot = k >> r.log_lanes;
    const float v = slot == 0 ? value[0] : slot == 1 ? value[1] : slot == 2 ? value[2] : value[3];
    sum = sum + __shfl(v, first + (k & ((1 << r.log_lanes) - 1)));
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int k = (q << r.log_lanes) + p;
    if (store && k < r.top_k) {
      idx_row[k] = taken[q];
      gates_row[k] = sigmoid ? (value[q] / (sum + 1e-9f)) * r.rsf : value[q] / sum;
    }
  }
}

}  // namespace hmoe
