// Router entries with the selection limited to groups (route_groups.h): in the router's launch
// for up to eight experts a token, from its logits for more, and from given logits.  (As a launch
// behind the logits one token on 64 experts takes 16.1 us against 14.5, 4096 on 256 82.6 against
// 75.0; without groups the router's launch takes 16.3 and 77.1.)
#include "router_kernels.h"

namespace hmoe {
namespace {

// Selection and gates among the experts of the best groups from given logits.  A wave takes 64
// >> log_lanes tokens, whose logits, one run of memory, go through LDS, and the biases: a lane
// reads E of each one after another (four words more every 32, so that lanes 32 words apart read
// different banks).  WIDE: the lanes' reads 16 bytes at a time, `wide_in`: the loads from memory.
template <int E, int L, bool WIDE>
__global__ __launch_bounds__(256) void select_groups_kernel(const float* __restrict__ logits,
                                                            const float* __restrict__ bias, int64_t tokens,
                                                            GroupRule r, bool wide_in,
                                                            int32_t* __restrict__ top_idx,
                                                            float* __restrict__ gates) {
  extern __shared__ __attribute__((aligned(16))) float stage[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int per_wave = 64 >> r.log_lanes;
  const int n = r.n_experts;
  const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * 4 + wave) * per_wave;
  if (t0 >= tokens) return;  // uniform per wave; no barrier follows
  const int count = static_cast<int>(tokens - t0 < per_wave ? tokens - t0 : per_wave) * n;
  float* mine = stage + wave * (group_stage_words(per_wave * n) + group_stage_words(n));
  float* biases = mine + group_stage_words(per_wave * n);
  const float* src = logits + t0 * n;
  const auto park = [&](const float* from, float* to, int words) __attribute__((always_inline)) {
    int done = 0;
    if (wide_in) {  // uniform
      done = words & ~3;
      for (int i = lane * 4; i < done; i += 256)
        *reinterpret_cast<f32x4*>(to + i + (i >> 5) * 4) = *reinterpret_cast<const f32x4*>(from + i);
    }
    if (done < words)  // uniform
      for (int i = done + lane; i < words; i += 64) to[i + (i >> 5) * 4] = from[i];
  };
  park(src, mine, count);
  if (bias != nullptr) {
    park(bias, biases, n);
  } else if (r.mode == HMOE_ROUTE_SIGMOID_BIAS) {
    for (int i = lane; i < n; i += 64) biases[i + (i >> 5) * 4] = 0.0f;
  }
  const int64_t tok = t0 + (lane >> r.log_lanes);
  const bool store = tok < tokens;
  const int row = store ? static_cast<int>(tok - t0) * n : 0;
  // (a wave's LDS accesses run in their order)
  asm volatile("" ::: "memory");
  const auto read = [&](const float* from, int first, float (&v)[E]) __attribute__((always_inline)) {
    if constexpr (WIDE) {
#pragma unroll
      for (int j = 0; j < E; j += 4) {
        const int i = first + j;
        const f32x4 w = *reinterpret_cast<const f32x4*>(from + i + (i >> 5) * 4);
#pragma unroll
        for (int q = 0; q < 4; ++q) v[j + q] = w[q];
      }
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = from[first + j + ((first + j) >> 5) * 4];
    }
  };
  const auto run = [&](int e, float (&l)[E], float (&b)[E]) __attribute__((always_inline)) {
    read(mine, row + e, l);
    if (r.mode == HMOE_ROUTE_SIGMOID_BIAS) read(biases, e, b);
  };
  const auto get = [&](int e) __attribute__((always_inline)) { return mine[row + e + ((row + e) >> 5) * 4]; };
  const int64_t tq = store ? tok : t0;
  select_in_groups<E, L>(run, get, r, store, top_idx + tq * r.top_k, gates + tq * r.top_k);
}

template <int E>
void launch_select_groups(const float* logits, const float* bias, int64_t tokens, int n_experts, int n_groups,
                          int top_groups, int top_k, int mode, float rsf, int32_t* top_idx, float* gates,
                          hipStream_t s) {
  const GroupRule r = group_rule(n_experts, n_groups, top_groups, top_k, mode, rsf, E);
  const int per_wave = 64 >> r.log_lanes;
  const size_t lds =
      static_cast<size_t>(4) * (group_stage_words(per_wave * n_experts) + group_stage_words(n_experts)) * sizeof(float);
  const dim3 grid(static_cast<unsigned>(ceil_div(tokens, 4 * per_wave)));
  // (a wave's logits start a multiple of per_wave * n_experts words on)
  const bool wide_in =
      per_wave * n_experts % 4 == 0 && aligned_to(logits, 16) && (bias == nullptr || aligned_to(bias, 16));
  const auto launch = [&](auto L, auto WIDE) {
    hipLaunchKernelGGL((select_groups_kernel<E, decltype(L)::value, decltype(WIDE)::value>), grid, dim3(256), lds, s,
                       logits, bias, tokens, r, wide_in, top_idx, gates);
  };
  const auto with_list = [&](auto L) {
    if (r.size % 4 == 0) launch(L, IntC<1>());
    else launch(L, IntC<0>());
  };
  if (top_k <= kList) with_list(IntC<kList>());
  else if (top_k <= kLongList) with_list(IntC<kLongList>());
  else with_list(IntC<kLongestList>());
}

// E: as many keys a lane as leave a token eight lanes and more (16384 tokens on 256 experts in
// eight groups, E 8, 16 and 32: 15.8, 11.0 and 12.3 us).
void select_groups(const float* logits, const float* bias, int64_t tokens, int n_experts, int n_groups,
                   int top_groups, int top_k, int mode, float rsf, int32_t* top_idx, float* gates, hipStream_t s) {
  const auto run = [&](auto E) {
    launch_select_groups<decltype(E)::value>(logits, bias, tokens, n_experts, n_groups, top_groups, top_k, mode, rsf,
                                             top_idx, gates, s);
  };
  const int size = n_experts / n_groups;
  int groups = 1;
  while (groups < n_groups) groups *= 2;
  const int keys = groups >= 8 ? size : (size * groups + 7) / 8;  // for one lane
  if (keys <= 8) run(IntC<8>());
  else run(IntC<16>());
}

int validate_groups(int64_t tokens, int n_experts, int top_k, int mode, int n_groups, int top_groups) {
  // (a launch has fewer than 2^32 threads: 64 a token for the selection, in workgroups of four
  // tokens and more, and for the logits of more than 240 experts, in workgroups of sixteen)
  HMOE_REQUIRE(tokens <= (int64_t(1) << 26) - 16, "router: tokens must be at most 2^26 - 16 with groups (got %lld)",
               (long long)tokens);
  HMOE_REQUIRE(n_groups >= 1 && n_groups <= kMaxGroups && n_experts % n_groups == 0,
               "router: n_groups must divide n_experts and be in [1, %d] (got %d, n_experts %d)", kMaxGroups, n_groups,
               n_experts);
  HMOE_REQUIRE(top_groups >= 1 && top_groups <= n_groups, "router: top_groups must be in [1, n_groups] (got %d of %d)",
               top_groups, n_groups);
  const int size = n_experts / n_groups;
  HMOE_REQUIRE(top_groups == n_groups || mode == HMOE_ROUTE_SOFTMAX || size >= 2,
               "router: a group's score is the sum of two: groups need two experts (n_experts %d in %d groups)",
               n_experts, n_groups);
  HMOE_REQUIRE(top_k <= top_groups * size, "router: top_k %d of the %d experts that top_groups %d leave", top_k,
               top_groups * size, top_groups);
  return HMOE_OK;
}

}  // namespace
}  // namespace hmoe

extern "C" int hmoe_router_grouped(const void* x, int x_dtype, const void* router_w, int w_dtype, const float* bias,
                                   int64_t tokens, int d_model, int n_experts, int top_k, int mode,
                                   float routed_scaling_factor, int n_groups, int top_groups, float* logits,
                                   int32_t* top_idx, float* gates, hmoe_stream_t stream) {
  using namespace hmoe;
  if (int rc = validate_routing(tokens, n_experts, top_k, mode)) return rc;
  if (int rc = validate_groups(tokens, n_experts, top_k, mode, n_groups, top_groups)) return rc;
  if (top_groups == n_groups)  // every expert is left
    return hmoe_router(x, x_dtype, router_w, w_dtype, bias, tokens, d_model, n_experts, top_k, mode,
                       routed_scaling_factor, logits, top_idx, gates, stream);
  HMOE_REQUIRE(d_model >= 8 && d_model % 8 == 0,
               "router_grouped: d_model must be a positive multiple of 8 (got %d)", d_model);
  HMOE_REQUIRE(x_dtype == HMOE_F32 || x_dtype == HMOE_BF16, "router_grouped: x dtype must be F32 or BF16");
  HMOE_REQUIRE(w_dtype == HMOE_F32 || w_dtype == HMOE_BF16, "router_grouped: weight dtype must be F32 or BF16");
  if (tokens == 0) return HMOE_OK;
  HMOE_REQUIRE(x && router_w && logits && top_idx && gates, "router_grouped: null pointer argument");
  const float* used_bias = mode == HMOE_ROUTE_SIGMOID_BIAS ? bias : nullptr;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (top_k <= kList) {
    XQuant with;
    with.to = kGroups;
    with.rule = group_rule(n_experts, n_groups, top_groups, top_k, mode, routed_scaling_factor,
                           n_experts <= 64 ? kGroupKeys<64> : kGroupKeys<256>);
    route_by_experts<true>(x_dtype, w_dtype, x, router_w, used_bias, tokens, d_model, n_experts, top_k, mode,
                           routed_scaling_factor, logits, top_idx, gates, s, with);
    return check_launch("hmoe_router_grouped");
  }
  // the logits (and the largest one's expert, which is written over), then the selection
  if (int rc = hmoe_router(x, x_dtype, router_w, w_dtype, nullptr, tokens, d_model, n_experts, 1, HMOE_ROUTE_SOFTMAX,
                           1.0f, logits, top_idx, gates, stream))
    return rc;
  select_groups(logits, used_bias, tokens, n_experts, n_groups, top_groups, top_k, mode, routed_scaling_factor, top_idx,
                gates, s);
  return check_launch("hmoe_router_grouped");
}

extern "C" int hmoe_router_grouped_from_logits(const float* logits, const float* bias, int64_t tokens, int n_experts,
                                               int top_k, int mode, float routed_scaling_factor, int n_groups,
                                               int top_groups, int32_t* top_idx, float* gates, hmoe_stream_t stream) {
  using namespace hmoe;
  if (int rc = validate_routing(tokens, n_experts, top_k, mode)) return rc;
  if (int rc = validate_groups(tokens, n_experts, top_k, mode, n_groups, top_groups)) return rc;
  if (top_groups == n_groups)
    return hmoe_router_from_logits(logits, bias, tokens, n_experts, top_k, mode, routed_scaling_factor, top_idx, gates,
                                   stream);
  if (tokens == 0) return HMOE_OK;
  HMOE_REQUIRE(logits && top_idx && gates, "router_grouped_from_logits: null pointer argument");
  select_groups(logits, mode == HMOE_ROUTE_SIGMOID_BIAS ? bias : nullptr, tokens, n_experts, n_groups, top_groups,
                top_k, mode, routed_scaling_factor, top_idx, gates, static_cast<hipStream_t>(stream));
  return check_launch("hmoe_router_grouped_from_logits");
}
