// Products of rows sorted by expert (or node type) with one matrix per expert.
//
// Rows offsets[e] .. offsets[e + 1] are those of expert e.  Product: out[r, :] = rows[r, :] W[e(r)], zeros for rows of no expert.
// Its gradient for the rows is the product of the output's gradient with the transposed matrices, the same kernel; that for the
// matrices is grad_W[e] = sum over the rows r of e of rows[r, :]^T grad[r, :].
#include <type_traits>

#include "group_plan.cuh"
#include "launch.cuh"
#include "row_values.cuh"
#include "scan.cuh"

namespace gsb {

constexpr int kTile = 64, kDepth = 16, kThreads = 256;

template <class T>
__device__ __forceinline__ float as_float(T v) {
  return (float)v;
}

// acc[4][4] += sum over l < depth of A(i, l) * B(l, j) for the tile's rows i < height and columns j < width.
template <class T, class Acc>
__device__ __forceinline__ void tile_product(Acc (&acc)[4][4], const T* a, i64 a_i, i64 a_l, u32 height, const T* b, i64 b_l, i64 b_j, u32 width,
                                             i64 depth, Acc (&sa)[kDepth][kTile + 1], Acc (&sb)[kDepth][kTile + 1]) {
  const int t = threadIdx.x, ti = t / 16, tj = t % 16;
  for (i64 l0 = 0; l0 < depth; l0 += kDepth) {
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kTile * kDepth / kThreads; ++s) {
      const int at = s * kThreads + t;
      const int i = at / kDepth, l = at % kDepth;
      sa[l][i] = (u32)i < height && l0 + l < depth ? (Acc)as_float(a[i * a_i + (l0 + l) * a_l]) : (Acc)0;
      sb[l][i] = (u32)i < width && l0 + l < depth ? (Acc)as_float(b[i * b_j + (l0 + l) * b_l]) : (Acc)0;
    }
    __syncthreads();
#pragma unroll
    for (int l = 0; l < kDepth; ++l)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += sa[l][ti * 4 + i] * sb[l][tj * 4 + j];
  }
}

struct ProductArgs {
  Groups groups;
  const void *rows, *weights;
  i64 rows_stride, w_expert, w_k, w_n;
  u32 k, n;
  const float *row_scales, *weight_scales;  // of 8-bit operands
};

template <class T, class Out>
__global__ void __launch_bounds__(kThreads) k_product(const ProductArgs a, Out* __restrict__ out) {
  using Acc = std::conditional_t<std::is_same<T, signed char>::value, int, float>;
  __shared__ PlanTable plan;
  __shared__ Acc sa[kDepth][kTile + 1], sb[kDepth][kTile + 1];
  await_previous();
  const Groups& g = a.groups;
  make_plan<kThreads>(plan, g, kTile, 0);
  const u32 columns = (a.n + kTile - 1) / kTile;
  const u64 tiles = (u64)plan.tile[g.experts] * columns;
  const int ti = threadIdx.x / 16 * 4, tj = threadIdx.x % 16 * 4;
  for (u64 t = blockIdx.x; t < tiles; t += gridDim.x) {
    const u32 row_tile = (u32)(t / columns), n0 = (u32)(t % columns) * kTile;
    const int e = expert_of_tile(plan, g.experts, row_tile);
    const u32 r0 = plan.begin[e] + (row_tile - plan.tile[e]) * kTile, height = min((u32)kTile, rows_end(plan, e) - r0);
    Acc acc[4][4] = {};
    tile_product<T, Acc>(acc, (const T*)a.rows + (i64)r0 * a.rows_stride, a.rows_stride, 1, height,
                         (const T*)a.weights + (i64)(g.first + e) * a.w_expert + (i64)n0 * a.w_n, a.w_k, a.w_n, min((u32)kTile, a.n - n0), a.k, sa, sb);
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 4; ++j) {
        if ((u32)(ti + i) >= height || n0 + tj + j >= a.n) continue;
        const u32 r = r0 + ti + i, c = n0 + tj + j;
        float v = (float)acc[i][j];
        if (a.row_scales) v = v * a.row_scales[r] * a.weight_scales[(i64)(g.first + e) * a.n + c];
        out[(i64)r * a.n + c] = from_float<Out>(v);
      }
  }
  // rows of no expert
  const i64 step = (i64)gridDim.x * kThreads, at = (i64)blockIdx.x * kThreads + threadIdx.x;
  if (g.first == 0)
    for (i64 i = at; i < (i64)plan.begin[0] * a.n; i += step) out[i] = from_float<Out>(0.f);
  if (g.first + g.experts == g.all)
    for (i64 i = (i64)plan.begin[g.experts] * a.n + at; i < (i64)g.num_rows * a.n; i += step) out[i] = from_float<Out>(0.f);
}

template <class T>
__global__ void __launch_bounds__(kThreads) k_grad_weights(const Groups g, const T* __restrict__ rows, i64 rows_stride, u32 k,
                                                           const T* __restrict__ grad, i64 grad_stride, u32 n, T* __restrict__ out) {
  __shared__ float sa[kDepth][kTile + 1], sb[kDepth][kTile + 1];
  await_previous();
  const u32 columns = (n + kTile - 1) / kTile, heights = (k + kTile - 1) / kTile;
  const u64 tiles = (u64)g.experts * columns * heights;
  const int ti = threadIdx.x / 16 * 4, tj = threadIdx.x % 16 * 4;
  for (u64 t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int e = (int)(t / ((u64)columns * heights));
    const u32 rest = (u32)(t % ((u64)columns * heights)), k0 = rest / columns * kTile, n0 = rest % columns * kTile;
    const i64 from = __ldg(g.offsets + e), to = __ldg(g.offsets + e + 1);
    if ((from < 0 || to < from || to > (i64)g.num_rows) && threadIdx.x == 0 && rest == 0) raise_error(g.counters, GSB_ERR_INDEX_RANGE, g.first + e);
    const u32 begin = clamped_offset(g, e), end = max(begin, clamped_offset(g, e + 1));
    const u32 height = min((u32)kTile, k - k0), width = min((u32)kTile, n - n0);
    float acc[4][4] = {};
    tile_product<T, float>(acc, rows + (i64)begin * rows_stride + k0, 1, rows_stride, height, grad + (i64)begin * grad_stride + n0, grad_stride, 1,
                           width, end - begin, sa, sb);
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 4; ++j)
        if ((u32)(ti + i) < height && (u32)(tj + j) < width)
          out[(i64)(g.first + e) * k * n + (i64)(k0 + ti + i) * n + n0 + tj + j] = from_float<T>(acc[i][j]);
  }
}

static int check_product(i64 num_rows, i64 k, i64 n, i64 num_experts, i64 rows_stride, const int64_t* offsets) {
  GSB_REQUIRE(num_rows >= 0 && num_rows < ((i64)1 << 31) && k >= 1 && k <= GSB_MAX_ROW_LEN && n >= 1 && n <= GSB_MAX_ROW_LEN && num_experts >= 1 &&
                  num_experts <= GSB_MAX_EXPERTS && rows_stride >= 0,
              GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(offsets && aligned_to(8, offsets), GSB_ERR_INVALID_ARGUMENT);
  return GSB_OK;
}

// One launch per kPlanExperts experts.
template <class F>
static int by_experts(gsb_ctx* ctx, i64 num_experts, i64 num_rows, const int64_t* offsets, F launch) {
  for (i64 first = 0; first < num_experts; first += kPlanExperts) {
    const int some = (int)min((i64)kPlanExperts, num_experts - first);
    const int st = launch(Groups{offsets + first, (int)first, some, (int)num_experts, (u32)num_rows, ctx_counters(ctx)});
    if (st != GSB_OK) return st;
  }
  return GSB_OK;
}

}  // namespace gsb

using namespace gsb;

extern "C" int64_t gsb_expert_product_workspace(const void* rows, int dtype, int64_t num_rows, int64_t k, int64_t rows_stride, const void* weights,
                                                int64_t weights_expert_stride, int64_t weights_k_stride, int64_t weights_n_stride, int64_t n,
                                                int64_t num_experts) {
  return 0;
}

extern "C" int gsb_expert_product(gsb_ctx* ctx, void* stream_, const void* rows, int dtype, int64_t num_rows, int64_t k, int64_t rows_stride,
                                  const void* weights, int64_t weights_expert_stride, int64_t weights_k_stride, int64_t weights_n_stride, int64_t n,
                                  const int64_t* offsets, int64_t num_experts, void* out, void* workspace, int64_t workspace_bytes) {
  GSB_ENTER(ctx);
  const int st = check_product(num_rows, k, n, num_experts, rows_stride, offsets);
  if (st != GSB_OK) return st;
  const int size = value_bytes(dtype);
  GSB_REQUIRE(size != 0 && weights_expert_stride >= 0 && weights_k_stride >= 0 && weights_n_stride >= 0, GSB_ERR_INVALID_ARGUMENT);
  if (num_rows == 0) return GSB_OK;
  GSB_REQUIRE(rows && weights && out && aligned_to(size, (const char*)rows, (const char*)weights, (const char*)out), GSB_ERR_INVALID_ARGUMENT);
  cudaStream_t stream = (cudaStream_t)stream_;
  return by_experts(ctx, num_experts, num_rows, offsets, [&](const Groups& g) {
    ScopedKernelTimer timer(ctx, KID_EXPERT_PRODUCT, stream);
    const ProductArgs a{g, rows, weights, rows_stride, weights_expert_stride, weights_k_stride, weights_n_stride, (u32)k, (u32)n, nullptr, nullptr};
    if (dtype == GSB_F32) launch_behind(stream, k_product<float, float>, kNumSMs * 4, kThreads, a, (float*)out);
    else if (dtype == GSB_F16) launch_behind(stream, k_product<__half, __half>, kNumSMs * 4, kThreads, a, (__half*)out);
    else launch_behind(stream, k_product<__nv_bfloat16, __nv_bfloat16>, kNumSMs * 4, kThreads, a, (__nv_bfloat16*)out);
    GSB_LAUNCH_OK();
    return (int)GSB_OK;
  });
}

extern "C" int64_t gsb_expert_product_grad_workspace(const void* rows, int dtype, int64_t num_rows, int64_t k, int64_t rows_stride, const void* grad,
                                                     int64_t n, int64_t grad_stride, int64_t num_experts) {
  return 0;
}

extern "C" int gsb_expert_product_grad(gsb_ctx* ctx, void* stream_, const void* rows, int dtype, int64_t num_rows, int64_t k, int64_t rows_stride,
                                       const void* grad, int64_t n, int64_t grad_stride, const int64_t* offsets, int64_t num_experts, void* out,
                                       void* workspace, int64_t workspace_bytes) {
  GSB_ENTER(ctx);
  const int st = check_product(num_rows, k, n, num_experts, rows_stride, offsets);
  if (st != GSB_OK) return st;
  const int size = value_bytes(dtype);
  GSB_REQUIRE(size != 0 && grad_stride >= 0 && out && ((rows && grad) || num_rows == 0), GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(aligned_to(size, (const char*)rows, (const char*)grad, (const char*)out), GSB_ERR_INVALID_ARGUMENT);
  cudaStream_t stream = (cudaStream_t)stream_;
  return by_experts(ctx, num_experts, num_rows, offsets, [&](const Groups& g) {
    ScopedKernelTimer timer(ctx, KID_EXPERT_PRODUCT, stream);
    with_unit(dtype, size, [&](auto value, auto) {
      typedef decltype(value) T;
      launch_behind(stream, k_grad_weights<T>, kNumSMs * 4, kThreads, g, (const T*)rows, rows_stride, (u32)k, (const T*)grad, grad_stride, (u32)n,
                    (T*)out);
    });
    GSB_LAUNCH_OK();
    return (int)GSB_OK;
  });
}

extern "C" int gsb_expert_product_int8(gsb_ctx* ctx, void* stream_, const int8_t* values, int64_t num_rows, int64_t k, int64_t values_stride,
                                       const float* scales, const int8_t* weight_values, int64_t weight_expert_stride, int64_t weight_n_stride,
                                       const float* weight_scales, int64_t n, const int64_t* offsets, int64_t num_experts, void* out, int out_dtype) {
  GSB_ENTER(ctx);
  const int st = check_product(num_rows, k, n, num_experts, values_stride, offsets);
  if (st != GSB_OK) return st;
  const int size = value_bytes(out_dtype);
  GSB_REQUIRE(size != 0 && k <= GSB_MAX_INT8_ROW_LEN && weight_expert_stride >= 0 && weight_n_stride >= 0, GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(aligned_to(16, values, weight_values) && values_stride % 16 == 0 && weight_expert_stride % 16 == 0 && weight_n_stride % 16 == 0,
              GSB_ERR_INVALID_ARGUMENT);
  if (num_rows == 0) return GSB_OK;
  GSB_REQUIRE(values && scales && weight_values && weight_scales && out && aligned_to(4, scales, weight_scales) && aligned_to(size, (const char*)out),
              GSB_ERR_INVALID_ARGUMENT);
  cudaStream_t stream = (cudaStream_t)stream_;
  return by_experts(ctx, num_experts, num_rows, offsets, [&](const Groups& g) {
    ScopedKernelTimer timer(ctx, KID_EXPERT_PRODUCT, stream);
    const ProductArgs a{g, values, weight_values, values_stride, weight_expert_stride, 1, weight_n_stride, (u32)k, (u32)n, scales, weight_scales};
    with_unit(out_dtype, size, [&](auto value, auto) {
      typedef decltype(value) Out;
      launch_behind(stream, k_product<signed char, Out>, kNumSMs * 4, kThreads, a, (Out*)out);
    });
    GSB_LAUNCH_OK();
    return (int)GSB_OK;
  });
}
