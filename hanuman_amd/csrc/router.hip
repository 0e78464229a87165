// Router entries with the plain selection (router_kernels.h), and selection from given logits.
#include "router_kernels.h"

namespace hmoe {
namespace {

// One wave per token: selection and gates from given logits.
// Tokens per wave (their reduction chains would interleave); one measured
// fastest once the reductions moved off the LDS permutes (4: 24.5 against
// 22.8 us at 32768 tokens, 64 experts, top-8).
constexpr int kSelTok = 1;

template <int EPL>
__global__ __launch_bounds__(256) void select_kernel(const float* __restrict__ logits,
                                                     const float* __restrict__ bias, int64_t tokens,
                                                     int n_experts, int top_k, int mode, float rsf,
                                                     int32_t* __restrict__ top_idx,
                                                     float* __restrict__ gates) {
  const int lane = threadIdx.x & 63;
  const int64_t tok0 = (static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6)) * kSelTok;
  if (tok0 >= tokens) return;
  float bv[EPL];
  load_bias(bv, mode == HMOE_ROUTE_SIGMOID_BIAS ? bias : nullptr, lane, 64, n_experts);
  float l[kSelTok][EPL];
  bool st[kSelTok];
  int32_t* ti[kSelTok];
  float* gt[kSelTok];
#pragma unroll
  for (int q = 0; q < kSelTok; ++q) {
    st[q] = tok0 + q < tokens;
    const int64_t tq = st[q] ? tok0 + q : tok0;  // a token past the end repeats the first
    ti[q] = top_idx + tq * top_k;
    gt[q] = gates + tq * top_k;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int e = lane + 64 * j;
      l[q][j] = e < n_experts ? logits[tq * n_experts + e] : 0.0f;
    }
  }
  select_and_gate<EPL, kSelTok>(l, st, bv, n_experts, top_k, mode, rsf, ti, gt);
}

// Selection and gates from given logits for up to 64 experts, eight tokens
// per wave (lane group lane / 8 one token, lane p its experts 8p .. 8p + 7).
__global__ __launch_bounds__(256) void select_kernel_g8(const float* __restrict__ logits,
                                                        const float* __restrict__ bias,
                                                        int64_t tokens, int n_experts, int top_k,
                                                        int mode, float rsf,
                                                        int32_t* __restrict__ top_idx,
                                                        float* __restrict__ gates) {
  const int lane = threadIdx.x & 63;
  const int p = lane & 7;
  const int64_t tok0 = (static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6)) * 8;
  if (tok0 >= tokens) return;  // uniform per wave
  const int64_t tok = tok0 + (lane >> 3);
  const bool st = tok < tokens;
  const int64_t tq = st ? tok : tokens - 1;
  float bv[8];
  load_bias(bv, mode == HMOE_ROUTE_SIGMOID_BIAS ? bias : nullptr, p * 8, 1, n_experts);
  float l[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int e = p * 8 + j;
    l[j] = e < n_experts ? logits[tq * n_experts + e] : 0.0f;
  }
  select_group8<8>(l, st, bv, n_experts, top_k, mode, rsf, top_idx + tq * top_k,
                   gates + tq * top_k);
}

}  // namespace
}  // namespace hmoe

extern "C" int hmoe_router(const void* x, int x_dtype, const void* router_w, int w_dtype,
                           const float* bias, int64_t tokens, int d_model, int n_experts,
                           int top_k, int mode, float routed_scaling_factor, float* logits,
                           int32_t* top_idx, float* gates, hmoe_stream_t stream) {
  using namespace hmoe;
  if (int rc = validate_routing(tokens, n_experts, top_k, mode)) return rc;
  HMOE_REQUIRE(d_model >= 8 && d_model % 8 == 0,
               "router: d_model must be a positive multiple of 8 (got %d)", d_model);
  HMOE_REQUIRE(x_dtype == HMOE_F32 || x_dtype == HMOE_BF16, "router: x dtype must be F32 or BF16");
  HMOE_REQUIRE(w_dtype == HMOE_F32 || w_dtype == HMOE_BF16, "router: weight dtype must be F32 or BF16");
  if (tokens == 0) return HMOE_OK;
  HMOE_REQUIRE(x && router_w && logits && top_idx && gates, "router: null pointer argument");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const float rsf = routed_scaling_factor;
  route_by_experts<false>(x_dtype, w_dtype, x, router_w, bias, tokens, d_model, n_experts, top_k, mode, rsf, logits,
                   top_idx, gates, s, XQuant());
  return check_launch("hmoe_router");
}

extern "C" int hmoe_router_quant_fp8(const void* x, int x_dtype, const void* router_w, int w_dtype,
                                     const float* bias, int64_t tokens, int d_model, int n_experts,
                                     int top_k, int mode, float routed_scaling_factor,
                                     float* logits, int32_t* top_idx, float* gates, uint8_t* x_q,
                                     float* x_scale, hmoe_stream_t stream) {
  using namespace hmoe;
  if (int rc = validate_routing(tokens, n_experts, top_k, mode)) return rc;
  HMOE_REQUIRE(d_model >= 8 && d_model % 8 == 0,
               "router_quant_fp8: d_model must be a positive multiple of 8 (got %d)", d_model);
  HMOE_REQUIRE(x_dtype == HMOE_BF16, "router_quant_fp8: x dtype must be BF16");
  HMOE_REQUIRE(w_dtype == HMOE_F32 || w_dtype == HMOE_BF16,
               "router_quant_fp8: weight dtype must be F32 or BF16");
  if (tokens == 0) return HMOE_OK;
  HMOE_REQUIRE(x && router_w && logits && top_idx && gates && x_q && x_scale,
               "router_quant_fp8: null pointer argument");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const float rsf = routed_scaling_factor;
  const XQuant xq{kQuantE4m3, x_q, x_scale};
  route_by_experts<false>(x_dtype, w_dtype, x, router_w, bias, tokens, d_model, n_experts, top_k, mode, rsf, logits,
                   top_idx, gates, s, xq);
  return check_launch("hmoe_router_quant_fp8");
}

extern "C" int hmoe_router_quant_mxfp4(const void* x, int x_dtype, const void* router_w, int w_dtype,
                                       const float* bias, int64_t tokens, int d_model, int n_experts,
                                       int top_k, int mode, float routed_scaling_factor,
                                       float* logits, int32_t* top_idx, float* gates, uint8_t* x_q,
                                       uint8_t* x_exp, hmoe_stream_t stream) {
  using namespace hmoe;
  if (int rc = validate_routing(tokens, n_experts, top_k, mode)) return rc;
  HMOE_REQUIRE_CODE(d_model >= kMxBlock && d_model % kMxBlock == 0, HMOE_ERR_UNSUPPORTED,
                    "router_quant_mxfp4: d_model must be a multiple of 32 (got %d)", d_model);
  HMOE_REQUIRE(x_dtype == HMOE_BF16, "router_quant_mxfp4: x dtype must be BF16");
  HMOE_REQUIRE(w_dtype == HMOE_F32 || w_dtype == HMOE_BF16,
               "router_quant_mxfp4: weight dtype must be F32 or BF16");
  if (tokens == 0) return HMOE_OK;
  HMOE_REQUIRE(x && router_w && logits && top_idx && gates && x_q && x_exp,
               "router_quant_mxfp4: null pointer argument");
  HMOE_REQUIRE_ALIGNED("router_quant_mxfp4", 16, x, x_q);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const float rsf = routed_scaling_factor;
  const XQuant xq{kQuantMxfp4, x_q, x_exp};
  route_by_experts<false>(x_dtype, w_dtype, x, router_w, bias, tokens, d_model, n_experts, top_k, mode, rsf, logits,
                   top_idx, gates, s, xq);
  return check_launch("hmoe_router_quant_mxfp4");
}

extern "C" int hmoe_router_from_logits(const float* logits, const float* bias, int64_t tokens,
                                       int n_experts, int top_k, int mode,
                                       float routed_scaling_factor, int32_t* top_idx,
                                       float* gates, hmoe_stream_t stream) {
  using namespace hmoe;
  if (int rc = validate_routing(tokens, n_experts, top_k, mode)) return rc;
  if (tokens == 0) return HMOE_OK;
  HMOE_REQUIRE(logits && top_idx && gates, "router_from_logits: null pointer argument");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(ceil_div(tokens, 4 * kSelTok)));
  if (n_experts <= 64)
    hipLaunchKernelGGL(select_kernel_g8, dim3(static_cast<unsigned>(ceil_div(tokens, 32))), dim3(256), 0, s,
                       logits, bias, tokens, n_experts, top_k, mode, routed_scaling_factor, top_idx, gates);
  else if (n_experts <= 128)
    hipLaunchKernelGGL(select_kernel<2>, grid, dim3(256), 0, s, logits, bias, tokens, n_experts, top_k, mode, routed_scaling_factor, top_idx, gates);
  else
    hipLaunchKernelGGL(select_kernel<4>, grid, dim3(256), 0, s, logits, bias, tokens, n_experts, top_k, mode, routed_scaling_factor, top_idx, gates);
  return check_launch("hmoe_router_from_logits");
}
