// Root-mean-square norm with the residual's addition (the block around model/moe.py:170;
// model/transformer.py:14-24 has the norm), with an output in 8 bits with scales:
//
//   s = rnd(x + r),   rstd = (sum_d s_d^2 / D + eps)^(-1/2),   y = rnd(s rstd w),
//
// and the codes and scale of the rounded y (e4m3 or int8 per row).  s is rounded to the
// residual's type first and the norm is the rounded sum's, since that is what the next
// block adds to and what the gradient sees.  Sums are float32, in a fixed order.
//
// Gradients, for cotangents dy of y and ds of s, with n = s rstd:
//
//   dx = dr = ds + rstd (dy w - n mean_d(dy w n)),   dw = sum_t dy n.
//
// All of it is bound by memory: a row is read once and kept in registers, from the addition
// through the norm to the codes, or from the dot product to dx and dw's part.  (As launches of
// their own addition, norm and quantisation would read and write 1.4 times the bytes.)
#include <algorithm>

#include "quant_i8.h"
#include "quant_mxfp4.h"
#include "rows.h"

namespace hmoe {
namespace {

struct NoResidual {};

struct Values8 {
  const float* v;
  __device__ __forceinline__ float get(int i) const { return v[i]; }
};

template <typename TX, typename TR>
struct SumType {
  typedef TR type;
};
template <typename TX>
struct SumType<TX, NoResidual> {
  typedef TX type;
};

// NT threads a row, C chunks of eight values each.  All loads of a row are issued before the
// first is used, past the caches' replacement (a row is not read again).  16384 x 2048 in bf16,
// with a residual and e4m3 codes: 51 us for 302 MB (6.0 TB/s, more than a copy's 4.9: half of
// the 134 MB that are read still lie in the 256 MB cache); int8 codes the same.  One row: 2.6 us,
// a chain of one load, two reductions and a store.
template <typename TX, typename TR, typename TY, int NT, int C>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void add_rms_norm_kernel(
    const TX* __restrict__ x, const TR* __restrict__ residual, const void* __restrict__ weight, bool weight_bf16,
    float eps, int64_t rows, int cols, typename SumType<TX, TR>::type* __restrict__ sum, TY* __restrict__ y,
    float* __restrict__ rstd_out, uint8_t* __restrict__ q, float* __restrict__ scale, int q_type) {
  constexpr int kThreads = NT < 256 ? 256 : NT;
  constexpr bool kAdd = !std::is_same<TR, NoResidual>::value;
  __shared__ float sum_part[2][NT / 64];
  __shared__ int32_t max_part[2][NT / 64];
  const int t = threadIdx.x % NT;
  const int chunks = cols / 8;
  int parity = 0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / NT) + threadIdx.x / NT; row < rows;
       row += static_cast<int64_t>(gridDim.x) * (kThreads / NT), parity ^= 1) {
    const int64_t r0 = row * cols;
    float v[C][8];
    float ss = 0.0f;
    Chunk8<TX> xv[C];
#pragma unroll
    for (int u = 0; u < C; ++u) {
      const int c = u * NT + t;
      xv[u].zero();
      if (c < chunks) xv[u].load_nt(x + r0 + c * 8);
    }
    if constexpr (kAdd) {
      Chunk8<TR> rv[C];
#pragma unroll
      for (int u = 0; u < C; ++u) {
        const int c = u * NT + t;
        rv[u].zero();
        if (c < chunks) rv[u].load_nt(residual + r0 + c * 8);
      }
#pragma unroll
      for (int u = 0; u < C; ++u) {
        const int c = u * NT + t;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = xv[u].get(i) + rv[u].get(i);
        if (c < chunks) round_store8(sum + r0 + c * 8, v[u]);
      }
    } else {
#pragma unroll
      for (int u = 0; u < C; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = xv[u].get(i);
    }
#pragma unroll
    for (int u = 0; u < C; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(v[u][i], v[u][i], ss);
    ss = row_sum<NT>(ss, sum_part[parity]);
    const float rstd = 1.0f / __builtin_sqrtf(ss / static_cast<float>(cols) + eps);
    if (rstd_out != nullptr && t == 0) rstd_out[row] = rstd;
#pragma unroll
    for (int u = 0; u < C; ++u) {
      const int c = u * NT + t;
      if (c < chunks) {
        float w[8];
        load8(weight, c * 8, weight_bf16, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = v[u][i] * rstd * w[i];
        round_store8(y + r0 + c * 8, v[u]);
      }
    }
    if (q == nullptr) continue;  // uniform
    if (q_type == HMOE_I8) {
      int32_t most = 0;
#pragma unroll
      for (int u = 0; u < C; ++u)
        if (u * NT + t < chunks) most = amax8_bits(v[u], most);
      const I8Scale s = i8_scale(row_max<NT>(most, max_part[parity]));
      if (t == 0) scale[row] = s.scale;
#pragma unroll
      for (int u = 0; u < C; ++u) {
        const int c = u * NT + t;
        if (c < chunks) *reinterpret_cast<uint2*>(q + r0 + c * 8) = i8_codes8(v[u], s);
      }
    } else {
      float most = 0.0f;
#pragma unroll
      for (int u = 0; u < C; ++u)
        if (u * NT + t < chunks)
#pragma unroll
          for (int i = 0; i < 8; ++i) most = amax_nan(most, v[u][i]);
      const int32_t bits = row_max<NT>(__float_as_int(most) & 0x7fffffff, max_part[parity]);
      float s, inv;
      e4m3_scales(__int_as_float(bits), s, inv);
      if (t == 0) scale[row] = s;
#pragma unroll
      for (int u = 0; u < C; ++u) {
        const int c = u * NT + t;
        if (c < chunks) *reinterpret_cast<uint2*>(q + r0 + c * 8) = quant8_e4m3(Values8{v[u]}, inv);
      }
    }
  }
}

// dw of few rows, 64 columns a workgroup: dy, s and rstd are all that it needs.  Runs of rows a
// stride apart, eight columns a thread, each summed on its own and the runs one after another.
template <typename TG, typename TS, int THREADS>
__device__ __forceinline__ void sum_columns(const TG* __restrict__ dy, const TS* __restrict__ s,
                                            const float* __restrict__ rstd, int rows, int cols,
                                            float* __restrict__ d_weight) {
  constexpr int kRuns = THREADS / 8;
  __shared__ float run[kRuns][65];
  const int c0 = blockIdx.x * 64, c = (threadIdx.x & 7) * 8;
  const int mine = threadIdx.x >> 3;
  float dw[8] = {};
  if (c0 + c < cols) {
#pragma unroll 4
    for (int row = mine; row < rows; row += kRuns) {
      Chunk8<TG> g;
      Chunk8<TS> v;
      g.load(dy + static_cast<int64_t>(row) * cols + c0 + c);
      v.load(s + static_cast<int64_t>(row) * cols + c0 + c);
      const float rs = rstd[row];
#pragma unroll
      for (int i = 0; i < 8; ++i) dw[i] = __builtin_fmaf(g.get(i), v.get(i) * rs, dw[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) run[mine][c + i] = dw[i];
  __syncthreads();
  if (threadIdx.x < 64 && c0 + static_cast<int>(threadIdx.x) < cols) {
    float total = run[0][threadIdx.x];
#pragma unroll 8
    for (int k = 1; k < kRuns; ++k) total += run[k][threadIdx.x];
    d_weight[c0 + threadIdx.x] = total;
  }
}

// Gradients.  A workgroup (NT 256 and more) or a wave (NT 64) takes rows a stride apart and
// keeps its columns' part of dw in registers; the parts are summed in their order by
// sum_parts_kernel.  16384 x 4096 in bf16: 82 us for 537 MB (6.5 TB/s; half of what is read
// lies in the 256 MB cache), and 4.7 for the parts; 2048 x 1536 in float32: 13 and 3.8, four rows
// one after another in each workgroup.  FEW: the first dw_groups workgroups sum dw's columns
// instead, beside the rows' (kFewRows).
template <typename TG, typename TS, int NT, int C, bool FEW>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void add_rms_norm_bwd_kernel(
    const TG* __restrict__ dy, const TS* __restrict__ s, const void* __restrict__ weight, bool weight_bf16,
    const float* __restrict__ rstd, const TS* __restrict__ d_sum, int64_t rows, int cols, TS* __restrict__ dx,
    float* __restrict__ dw_parts, unsigned dw_groups) {
  constexpr int kThreads = NT < 256 ? 256 : NT;
  if constexpr (FEW) {
    if (blockIdx.x < dw_groups) {  // uniform
      sum_columns<TG, TS, kThreads>(dy, s, rstd, static_cast<int>(rows), cols, dw_parts);
      return;
    }
  }
  __shared__ float part[2][NT / 64];
  const int t = threadIdx.x % NT;
  const int chunks = cols / 8;
  const int64_t first =
      static_cast<int64_t>(blockIdx.x - (FEW ? dw_groups : 0u)) * (kThreads / NT) + threadIdx.x / NT;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * (kThreads / NT);
  float dw[C][8] = {};
  // (a thread of 1024 has 128 registers: with four chunks, rows past 16384 values, the weight and
  // d_sum are read where they are used; 4000 x 32768 in bf16 312 us, held with the rest 488.  What is
  // left still passes 128 by 31 to 53 registers, and the loop spills: 1.46 times the bytes' time at a
  // copy's rate.  Two chunks, rows of 8193 to 16384 values, spill nothing.)
  constexpr bool kLean = NT == 1024 && C == 4;
  float w[kLean ? 1 : C][8];
  const auto weight8 = [&](int u, float (&v)[8]) __attribute__((always_inline)) {
    const int c = u * NT + t;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    if (c < chunks) load8(weight, c * 8, weight_bf16, v);
  };
  if constexpr (!kLean) {
#pragma unroll
    for (int u = 0; u < C; ++u) weight8(u, w[u]);
  }
  const auto take_weight = [&](int u, float (&v)[8]) __attribute__((always_inline)) {
    if constexpr (kLean) {
      weight8(u, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = w[u][i];
    }
  };
  int parity = 0;
  for (int64_t row = first; row < rows; row += stride, parity ^= 1) {
    const int64_t r0 = row * cols;
    Chunk8<TG> g[C];
    Chunk8<TS> sv[C], ds[kLean ? 1 : C];
#pragma unroll
    for (int u = 0; u < C; ++u) {
      const int c = u * NT + t;
      g[u].zero();
      sv[u].zero();
      if (!kLean) ds[u].zero();
      if (c < chunks) {
        g[u].load_nt(dy + r0 + c * 8);
        sv[u].load_nt(s + r0 + c * 8);
        if (!kLean && d_sum != nullptr) ds[u].load_nt(d_sum + r0 + c * 8);
      }
    }
    const float rs = rstd[row];
    float dot = 0.0f;
#pragma unroll
    for (int u = 0; u < C; ++u) {
      float wu[8];
      take_weight(u, wu);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = sv[u].get(i) * rs;
        dot = __builtin_fmaf(g[u].get(i) * wu[i], n, dot);
        dw[u][i] = __builtin_fmaf(g[u].get(i), n, dw[u][i]);
      }
    }
    const float mean = row_sum<NT>(dot, part[parity]) / static_cast<float>(cols);
#pragma unroll
    for (int u = 0; u < C; ++u) {
      const int c = u * NT + t;
      float d[8], wu[8];
      take_weight(u, wu);
      Chunk8<TS>& more = ds[kLean ? 0 : u];
      if constexpr (kLean) {
        more.zero();
        if (c < chunks && d_sum != nullptr) more.load_nt(d_sum + r0 + c * 8);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = sv[u].get(i) * rs;
        d[i] = more.get(i) + rs * (g[u].get(i) * wu[i] - n * mean);
      }
      if (c < chunks) round_store8(dx + r0 + c * 8, d);
    }
  }
  if (FEW || dw_parts == nullptr) return;
#pragma unroll
  for (int u = 0; u < C; ++u) {
    const int c = u * NT + t;
    if (c < chunks) round_store8(dw_parts + first * cols + c * 8, dw[u]);
  }
}

// out[c] = sum over the parts' rows in order: 32 columns a workgroup, 32 runs of rows, each
// summed on its own and the runs' sums then one after another.
__global__ __launch_bounds__(1024) void sum_parts_kernel(const float* __restrict__ parts, int n_parts, int cols,
                                                         float* __restrict__ out) {
  __shared__ float run[32][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31);
  const int g = threadIdx.x >> 5;
  const int lo = n_parts * g / 32, hi = n_parts * (g + 1) / 32;
  float sum = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int p = lo; p < hi; ++p) sum += parts[static_cast<int64_t>(p) * cols + c];
  }
  run[g][threadIdx.x & 31] = sum;
  __syncthreads();
  if (g == 0 && c < cols) {
    float total = run[0][threadIdx.x];
#pragma unroll
    for (int k = 1; k < 32; ++k) total += run[k][threadIdx.x];
    out[c] = total;
  }
}

// Parts that dw is summed in: rows of 1024 values and more are a workgroup's, and 512 of them
// keep the memory busy (16384 x 4096 in bf16: 88 us; 1024 parts 99, 384 91).  Shorter ones are
// a wave's, and are the more at a time the shorter they are (30000 x 512: 1024 parts 70 us, 2048
// 49; 100000 x 256: 1024 99, 2048 62, 4096 48; 200000 x 128 float32: 4096 102, 8192 107), and past
// 1024 of four rows at least (4000 x 1024: 1024 parts 13.6 us, 2048 16.8: the parts are read again).
constexpr int kBwdWaveCols = 1024;
constexpr int64_t kMaxParts = 4096;
// Up to so many rows dy and s are read again instead, by workgroups of the same launch, and no
// workspace is needed.  768 rows so and in parts, us: bf16 of 1536 columns 5.3 and 8.1, 4096 8.1 and
// 13.3, 8192 16 and 21, 32768 61 and 94; float32 8.1 and 9.2, 21.6 and 18.4, 28 and 31, 121 and 153.
// (1000 rows: 1536 columns of bf16 6.1 and 8.4, of float32 9.5 and 10.0, 4096 of float32 24.5 and 21.
// What the launch reads again grows with the rows, what the parts move does not.)
constexpr int64_t kFewRows = 768;
int64_t most_parts(int64_t rows, int cols) {
  if (cols > kBwdWaveCols || rows < kWaveRows) return 512;
  const int64_t most = std::max(int64_t(1024), std::min((int64_t(1) << 20) / cols, ceil_div(rows, 16) * 4));
  return most < kMaxParts ? most : kMaxParts;
}
struct BwdShape {
  unsigned grid;
  int parts;
};
BwdShape bwd_shape(int64_t rows, int cols) {
  BwdShape b{0, 0};
  with_row_form(rows, cols, kBwdWaveCols, [&](auto nt, auto) {
    constexpr int per_group = decltype(nt)::value == 64 ? 4 : 1;
    const int64_t most = most_parts(rows, cols) / per_group;
    const int64_t g = ceil_div(rows, per_group);
    b.grid = static_cast<unsigned>(g < most ? g : most);
    b.parts = static_cast<int>(b.grid) * per_group;
  });
  return b;
}

bool overlap(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + b_bytes && y < x + a_bytes;
}

bool float_type(int dtype) { return dtype == HMOE_F32 || dtype == HMOE_BF16; }

int check_rows(const char* what, int64_t rows, int cols) {
  // (2^40 rows: offsets stay in 64 bits, and no memory holds more)
  HMOE_REQUIRE(rows >= 0 && rows <= (int64_t(1) << 40), "%s: rows must be in [0, 2^40]", what);
  HMOE_REQUIRE_CODE(cols >= 8 && cols % 8 == 0 && cols <= kMaxRowCols, HMOE_ERR_UNSUPPORTED,
                    "%s: cols must be a multiple of 8 up to %d (got %d)", what, kMaxRowCols, cols);
  return HMOE_OK;
}

template <typename F>
void with_float_type(int dtype, F f) {
  if (dtype == HMOE_BF16) f(uint16_t{});
  else f(float{});
}

}  // namespace
}  // namespace hmoe

extern "C" int hmoe_add_rms_norm(const void* x, int x_dtype, const void* residual, int residual_dtype,
                                 const void* weight, int w_dtype, float eps, int64_t rows, int cols, void* sum,
                                 void* y, int y_dtype, float* rstd, void* q, int q_type, float* scale,
                                 hmoe_stream_t stream) {
  using namespace hmoe;
  const char* what = "add_rms_norm";
  if (int rc = check_rows(what, rows, cols)) return rc;
  HMOE_REQUIRE(float_type(x_dtype) && float_type(y_dtype) && float_type(w_dtype),
               "%s: x, weight and y dtypes must be F32 or BF16", what);
  HMOE_REQUIRE(residual == nullptr || float_type(residual_dtype), "%s: residual dtype must be F32 or BF16", what);
  HMOE_REQUIRE(q == nullptr || q_type == HMOE_FP8_E4M3 || q_type == HMOE_I8, "%s: q type must be FP8_E4M3 or I8",
               what);
  HMOE_REQUIRE(eps >= 0.0f, "%s: eps must not be negative", what);
  if (rows == 0) return HMOE_OK;
  HMOE_REQUIRE(x && weight && y && (q == nullptr) == (scale == nullptr) && (residual == nullptr) == (sum == nullptr),
               "%s: null pointer argument (sum goes with residual, scale with q)", what);
  HMOE_REQUIRE_ALIGNED(what, 16, x, residual, weight, sum, y);
  HMOE_REQUIRE_ALIGNED(what, 8, q);
  hipStream_t st = static_cast<hipStream_t>(stream);
  with_row_form(rows, cols, 2048, [&](auto nt, auto c) {
    constexpr int kNt = decltype(nt)::value, kC = decltype(c)::value;
    constexpr int kThreads = kNt < 256 ? 256 : kNt;
    with_float_type(x_dtype, [&](auto tx) {
      with_float_type(y_dtype, [&](auto ty) {
        typedef decltype(tx) TX;
        typedef decltype(ty) TY;
        const auto launch = [&](auto tr) {
          typedef decltype(tr) TR;
          hipLaunchKernelGGL((add_rms_norm_kernel<TX, TR, TY, kNt, kC>), dim3(row_grid(rows, kThreads / kNt)),
                             dim3(kThreads), 0, st, static_cast<const TX*>(x), static_cast<const TR*>(residual),
                             weight, w_dtype == HMOE_BF16, eps, rows, cols,
                             static_cast<typename SumType<TX, TR>::type*>(sum), static_cast<TY*>(y), rstd,
                             static_cast<uint8_t*>(q), scale, q_type);
        };
        if (residual == nullptr) launch(NoResidual{});
        else with_float_type(residual_dtype, launch);
      });
    });
  });
  return check_launch("hmoe_add_rms_norm");
}

extern "C" size_t hmoe_add_rms_norm_bwd_workspace_bytes(int64_t rows, int cols) {
  using namespace hmoe;
  if (rows <= 0 || cols <= 0) return 0;
  const int parts = rows <= kFewRows ? 1 : bwd_shape(rows, cols).parts;
  return parts > 1 ? static_cast<size_t>(parts) * cols * sizeof(float) : 0;
}

extern "C" int hmoe_add_rms_norm_bwd(const void* dy, int dy_dtype, const void* sum, int sum_dtype, const void* weight,
                                     int w_dtype, const float* rstd, const void* d_sum, int64_t rows, int cols,
                                     void* dx, float* d_weight, void* workspace, size_t workspace_bytes,
                                     hmoe_stream_t stream) {
  using namespace hmoe;
  const char* what = "add_rms_norm_bwd";
  if (int rc = check_rows(what, rows, cols)) return rc;
  HMOE_REQUIRE(float_type(dy_dtype) && float_type(sum_dtype) && float_type(w_dtype),
               "%s: dy, sum and weight dtypes must be F32 or BF16", what);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned columns = static_cast<unsigned>(ceil_div(cols, 32));
  if (rows == 0) {
    if (d_weight == nullptr) return HMOE_OK;
    hipLaunchKernelGGL(sum_parts_kernel, dim3(columns), dim3(1024), 0, st, static_cast<const float*>(nullptr), 0, cols,
                       d_weight);
    return check_launch("hmoe_add_rms_norm_bwd");
  }
  HMOE_REQUIRE(dy && sum && weight && rstd && dx, "%s: null pointer argument", what);
  HMOE_REQUIRE_ALIGNED(what, 16, dy, sum, weight, d_sum, dx, d_weight, workspace);
  const auto run = [&](auto few, unsigned grid, unsigned dw_groups, float* dw) {
    with_row_form(rows, cols, kBwdWaveCols, [&](auto nt, auto c) {
      constexpr int kNt = decltype(nt)::value, kC = decltype(c)::value;
      constexpr bool kFew = decltype(few)::value;
      // (few rows are a workgroup's each)
      if constexpr (!kFew || kNt > 64) {
        with_float_type(dy_dtype, [&](auto tg) {
          with_float_type(sum_dtype, [&](auto ts) {
            typedef decltype(tg) TG;
            typedef decltype(ts) TS;
            hipLaunchKernelGGL((add_rms_norm_bwd_kernel<TG, TS, kNt, kC, kFew>), dim3(grid),
                               dim3(kNt < 256 ? 256 : kNt), 0, st, static_cast<const TG*>(dy),
                               static_cast<const TS*>(sum), weight, w_dtype == HMOE_BF16, rstd,
                               static_cast<const TS*>(d_sum), rows, cols, static_cast<TS*>(dx), dw, dw_groups);
          });
        });
      }
    });
  };
  if (rows <= kFewRows) {
    static_assert(kFewRows < kWaveRows, "few rows are a workgroup's each");
    const unsigned groups = d_weight == nullptr ? 0u : static_cast<unsigned>(ceil_div(cols, 64));
    // dx may be written over sum or dy, which dw's columns read: then one launch behind the other
    const size_t values = static_cast<size_t>(rows) * cols, sum_size = sum_dtype == HMOE_BF16 ? 2 : 4;
    const size_t dx_bytes = values * sum_size;
    const bool over = overlap(dx, dx_bytes, sum, dx_bytes) ||
                      overlap(dx, dx_bytes, dy, values * (dy_dtype == HMOE_BF16 ? 2 : 4));
    if (over && groups > 0) {
      run(std::true_type{}, groups, groups, d_weight);
      run(std::true_type{}, static_cast<unsigned>(rows), 0u, nullptr);
    } else {
      run(std::true_type{}, groups + static_cast<unsigned>(rows), groups, d_weight);
    }
    return check_launch("hmoe_add_rms_norm_bwd");
  }
  const BwdShape b = bwd_shape(rows, cols);
  const size_t need = hmoe_add_rms_norm_bwd_workspace_bytes(rows, cols);
  HMOE_REQUIRE_CODE(d_weight == nullptr || need == 0 || (workspace && workspace_bytes >= need), HMOE_ERR_WORKSPACE,
                    "%s: workspace has %zu bytes, needs %zu", what, workspace ? workspace_bytes : size_t(0), need);
  float* parts = d_weight == nullptr ? nullptr : b.parts > 1 ? static_cast<float*>(workspace) : d_weight;
  run(std::false_type{}, b.grid, 0u, parts);
  if (d_weight != nullptr && b.parts > 1)
    hipLaunchKernelGGL(sum_parts_kernel, dim3(columns), dim3(1024), 0, st, static_cast<const float*>(parts), b.parts,
                       cols, d_weight);
  return check_launch("hmoe_add_rms_norm_bwd");
}
