// Rows sorted by expert (or by node type) and back.
//
// Order: slot s = t * K + k of token t wants expert e(s), or none (-1).  Slots are sorted by expert, stably; those without one
// come last.  place[s] is the row of slot s in that order, ~row (negative) for a slot without an expert.
// Spread:  rows[place[t, k], :] = w[t, k] * x[t, :] (w = 1 without weights), zeros in the rows of slots without an expert.
// Combine: out[t, :] = sum over k of w[t, k] * rows[place[t, k], :], slots without an expert left out.
// Combine's gradient: spread of the output's gradient for the rows, and for w[t, k] the product <grad[t, :], rows[place[t, k], :]>.
// Spread's gradient is a combine.  Sums are in float, in the order of k; each result is rounded once.
#include <type_traits>

#include "key_sort.cuh"
#include "row_values.cuh"
#include "scan.cuh"

namespace gsb {

constexpr int kRowThreads = 256;

// Weights of type float or of the rows' type, or none (all 1).
struct Weights {
  const void* p;
  int dtype;
};
__device__ __forceinline__ float weight_of(const Weights& w, i64 slot) {
  if (!w.p) return 1.f;
  if (w.dtype == GSB_F32) return __ldg((const float*)w.p + slot);
  if (w.dtype == GSB_F16) return __half2float(((const __half*)w.p)[slot]);
  return __bfloat162float(((const __nv_bfloat16*)w.p)[slot]);
}

struct RowArgs {
  i64 tokens, num_rows;
  int per_token, lanes;
  i64 units, token_stride, row_stride;  // in units
  const i64* place;
  Weights weights;
  i64* counters;
};

// Row of a slot, or ~row for a slot without an expert.  kNowhere: out of range, which is recorded, unless it is the row of a
// slot without an expert that a caller's shorter array does not have.
constexpr i64 kNowhere = (i64)1 << 62;
__device__ __forceinline__ i64 place_of(const RowArgs& a, i64 slot, bool report) {
  const i64 p = __ldg(a.place + slot);
  if ((u64)(p < 0 ? ~p : p) < (u64)a.num_rows) return p;
  if (report && (p >= 0 || ~p >= a.tokens * a.per_token)) raise_error(a.counters, GSB_ERR_INDEX_RANGE, slot);
  return kNowhere;
}

template <class T, int BYTES>
__global__ void __launch_bounds__(kRowThreads) k_spread_rows(const RowArgs a, const Unit<T, BYTES>* __restrict__ x,
                                                             Unit<T, BYTES>* __restrict__ rows) {
  const int lane = threadIdx.x & (a.lanes - 1);
  const i64 groups = (i64)gridDim.x * (kRowThreads / a.lanes);
  for (i64 t = ((i64)blockIdx.x * kRowThreads + threadIdx.x) / a.lanes; t < a.tokens; t += groups) {
    for (i64 j = lane; j < a.units; j += a.lanes) {
      const Unit<T, BYTES> v = load_unit_once(x + t * a.token_stride + j);
      for (int k = 0; k < a.per_token; ++k) {
        const i64 slot = t * a.per_token + k, p = place_of(a, slot, j == 0);
        if (p == kNowhere) continue;
        const float w = weight_of(a.weights, slot);
        Unit<T, BYTES> u;
#pragma unroll
        for (int q = 0; q < u.N; ++q) u.v[q] = p < 0 ? from_float<T>(0.f) : from_float<T>(to_float(v.v[q]) * w);
        store_unit(rows + (p < 0 ? ~p : p) * a.units + j, u);
      }
    }
  }
}

template <class T, int BYTES>
__global__ void __launch_bounds__(kRowThreads) k_combine_rows(const RowArgs a, const Unit<T, BYTES>* __restrict__ rows,
                                                              Unit<T, BYTES>* __restrict__ out) {
  const int lane = threadIdx.x & (a.lanes - 1);
  const i64 groups = (i64)gridDim.x * (kRowThreads / a.lanes);
  for (i64 t = ((i64)blockIdx.x * kRowThreads + threadIdx.x) / a.lanes; t < a.tokens; t += groups) {
    for (i64 j = lane; j < a.units; j += a.lanes) {
      float sum[Unit<T, BYTES>::N] = {};
#pragma unroll 4
      for (int k = 0; k < a.per_token; ++k) {
        const i64 slot = t * a.per_token + k, p = place_of(a, slot, j == 0);
        if (p < 0 || p == kNowhere) continue;
        const float w = weight_of(a.weights, slot);
        const Unit<T, BYTES> v = load_unit_once(rows + p * a.row_stride + j);
#pragma unroll
        for (int q = 0; q < v.N; ++q) sum[q] += to_float(v.v[q]) * w;
      }
      Unit<T, BYTES> u;
#pragma unroll
      for (int q = 0; q < u.N; ++q) u.v[q] = from_float<T>(sum[q]);
      store_unit(out + t * a.units + j, u);
    }
  }
}

template <class W>
__device__ __forceinline__ void store_weight(void* p, i64 slot, float v) {
  ((W*)p)[slot] = from_float<W>(v);
}

// A warp per slot.
template <class T, int BYTES>
__global__ void __launch_bounds__(kRowThreads) k_combine_grad(const RowArgs a, const Unit<T, BYTES>* __restrict__ grad,
                                                              const Unit<T, BYTES>* __restrict__ rows,
                                                              Unit<T, BYTES>* __restrict__ grad_rows, void* grad_weights) {
  const int lane = threadIdx.x & 31;
  const i64 warps = (i64)gridDim.x * (kRowThreads / 32), slots = a.tokens * a.per_token;
  for (i64 slot = ((i64)blockIdx.x * kRowThreads + threadIdx.x) / 32; slot < slots; slot += warps) {
    const i64 t = slot / a.per_token, p = place_of(a, slot, lane == 0);
    float dot = 0.f;
    if (p != kNowhere) {
      const float w = weight_of(a.weights, slot);
      for (i64 j = lane; j < a.units; j += 32) {
        Unit<T, BYTES> u;
        if (p >= 0) {
          const Unit<T, BYTES> g = load_unit(grad + t * a.token_stride + j);
          if (grad_weights) {
            const Unit<T, BYTES> v = load_unit_once(rows + p * a.row_stride + j);
#pragma unroll
            for (int q = 0; q < v.N; ++q) dot += to_float(v.v[q]) * to_float(g.v[q]);
          }
#pragma unroll
          for (int q = 0; q < u.N; ++q) u.v[q] = from_float<T>(to_float(g.v[q]) * w);
        } else {
#pragma unroll
          for (int q = 0; q < u.N; ++q) u.v[q] = from_float<T>(0.f);
        }
        if (grad_rows) store_unit(grad_rows + (p < 0 ? ~p : p) * a.units + j, u);
      }
    }
    if (!grad_weights) continue;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (lane != 0) continue;
    if (a.weights.dtype == GSB_F32) store_weight<float>(grad_weights, slot, dot);
    else if (a.weights.dtype == GSB_F16) store_weight<__half>(grad_weights, slot, dot);
    else store_weight<__nv_bfloat16>(grad_weights, slot, dot);
  }
}

static int check_rows(i64 tokens, i64 per_token, i64 row_len, int dtype, i64 stride, const void* place, const void* weights,
                      int weights_dtype) {
  GSB_REQUIRE(tokens >= 0 && per_token >= 1 && per_token < ((i64)1 << 31) && row_len >= 1 && row_len <= GSB_MAX_ROW_LEN &&
                  stride >= 0 && value_bytes(dtype) != 0,
              GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(tokens == 0 || place, GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(!weights || weights_dtype == dtype || weights_dtype == GSB_F32, GSB_ERR_INVALID_ARGUMENT);
  return GSB_OK;
}

static int group_lanes(i64 units) {
  int lanes = 1;
  while (lanes < 32 && lanes < units) lanes *= 2;
  return lanes;
}

}  // namespace gsb

using namespace gsb;

extern "C" int64_t gsb_expert_order_workspace(int64_t n, int64_t num_experts) {
  if (n < 0 || n >= ((int64_t)1 << 31) || num_experts < 1 || num_experts > GSB_MAX_EXPERTS) return GSB_ERR_INVALID_ARGUMENT;
  return (int64_t)key_sort_bytes(n, num_experts);
}

extern "C" int gsb_expert_order(gsb_ctx* ctx, void* stream_, const int64_t* experts, int64_t n, int64_t num_experts,
                                int64_t* out_offsets, int64_t* out_source, int64_t* out_place, void* workspace,
                                int64_t workspace_bytes) {
  GSB_ENTER(ctx);
  const int64_t need = gsb_expert_order_workspace(n, num_experts);
  GSB_REQUIRE(need >= 0 && out_offsets, GSB_ERR_INVALID_ARGUMENT);
  cudaStream_t stream = (cudaStream_t)stream_;
  if (n == 0) {
    GSB_CUDA_OK(cudaMemsetAsync(out_offsets, 0, (size_t)(num_experts + 1) * sizeof(int64_t), stream));
    return GSB_OK;
  }
  GSB_REQUIRE(experts && out_source && out_place && workspace, GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(workspace_bytes >= need, GSB_ERR_CAPACITY);
  SortCall call{KeySource{experts, n, num_experts, true, -1, ctx_counters(ctx)}, SORT_ORDER};
  call.offsets = out_offsets;
  call.order_source = out_source;
  call.place = out_place;
  ScopedKernelTimer timer(ctx, KID_KEY_SORT, stream);
  return key_sort(ctx, stream, call, workspace, nullptr);
}

extern "C" int gsb_expert_spread(gsb_ctx* ctx, void* stream_, const void* x, int dtype, int64_t tokens, int64_t per_token,
                                 int64_t row_len, int64_t x_stride, const int64_t* place, const void* weights,
                                 int weights_dtype, void* out_rows) {
  GSB_ENTER(ctx);
  const int st = check_rows(tokens, per_token, row_len, dtype, x_stride, place, weights, weights_dtype);
  if (st != GSB_OK) return st;
  if (tokens == 0) return GSB_OK;
  GSB_REQUIRE(x && out_rows, GSB_ERR_INVALID_ARGUMENT);
  cudaStream_t stream = (cudaStream_t)stream_;
  const int size = value_bytes(dtype);
  const int unit = unit_bytes(row_len * size, (u64)(uintptr_t)x | (u64)(uintptr_t)out_rows | (u64)(x_stride * size));
  ScopedKernelTimer timer(ctx, KID_EXPERT_ROWS, stream);
  with_unit(dtype, unit, [&](auto value, auto bytes) {
    typedef decltype(value) T;
    constexpr int B = decltype(bytes)::value;
    const i64 units = row_len * size / B;
    const RowArgs a{tokens, tokens * per_token, (int)per_token, group_lanes(units), units, x_stride * size / B, units,
                    place, Weights{weights, weights_dtype}, ctx_counters(ctx)};
    const int grid = (int)min((i64)kNumSMs * 32, (i64)grid_for(tokens * a.lanes, kRowThreads));
    k_spread_rows<T, B><<<grid, kRowThreads, 0, stream>>>(a, (const Unit<T, B>*)x, (Unit<T, B>*)out_rows);
  });
  GSB_LAUNCH_OK();
  return GSB_OK;
}

extern "C" int gsb_expert_combine(gsb_ctx* ctx, void* stream_, const void* rows, int dtype, int64_t num_rows, int64_t tokens,
                                  int64_t per_token, int64_t row_len, int64_t rows_stride, const int64_t* place,
                                  const void* weights, int weights_dtype, void* out) {
  GSB_ENTER(ctx);
  const int st = check_rows(tokens, per_token, row_len, dtype, rows_stride, place, weights, weights_dtype);
  if (st != GSB_OK) return st;
  GSB_REQUIRE(num_rows >= 0 && num_rows <= tokens * per_token, GSB_ERR_INVALID_ARGUMENT);
  if (tokens == 0) return GSB_OK;
  GSB_REQUIRE((rows || num_rows == 0) && out, GSB_ERR_INVALID_ARGUMENT);
  cudaStream_t stream = (cudaStream_t)stream_;
  const int size = value_bytes(dtype);
  const int unit = unit_bytes(row_len * size, (u64)(uintptr_t)rows | (u64)(uintptr_t)out | (u64)(rows_stride * size));
  ScopedKernelTimer timer(ctx, KID_EXPERT_ROWS, stream);
  with_unit(dtype, unit, [&](auto value, auto bytes) {
    typedef decltype(value) T;
    constexpr int B = decltype(bytes)::value;
    const i64 units = row_len * size / B;
    const RowArgs a{tokens, num_rows, (int)per_token, group_lanes(units), units, units, rows_stride * size / B,
                    place, Weights{weights, weights_dtype}, ctx_counters(ctx)};
    const int grid = (int)min((i64)kNumSMs * 32, (i64)grid_for(tokens * a.lanes, kRowThreads));
    k_combine_rows<T, B><<<grid, kRowThreads, 0, stream>>>(a, (const Unit<T, B>*)rows, (Unit<T, B>*)out);
  });
  GSB_LAUNCH_OK();
  return GSB_OK;
}

extern "C" int gsb_expert_combine_grad(gsb_ctx* ctx, void* stream_, const void* grad, int dtype, int64_t tokens,
                                       int64_t per_token, int64_t row_len, int64_t grad_stride, const void* rows,
                                       int64_t num_rows, int64_t rows_stride, const int64_t* place, const void* weights,
                                       int weights_dtype, void* out_grad_rows, void* out_grad_weights) {
  GSB_ENTER(ctx);
  const int st = check_rows(tokens, per_token, row_len, dtype, grad_stride, place, weights, weights_dtype);
  if (st != GSB_OK) return st;
  GSB_REQUIRE(num_rows >= 0 && num_rows <= tokens * per_token && rows_stride >= 0, GSB_ERR_INVALID_ARGUMENT);
  if (tokens == 0) return GSB_OK;
  GSB_REQUIRE(grad && (!out_grad_weights || (weights && (rows || num_rows == 0))), GSB_ERR_INVALID_ARGUMENT);
  cudaStream_t stream = (cudaStream_t)stream_;
  const int size = value_bytes(dtype);
  u64 addresses = (u64)(uintptr_t)grad | (u64)(uintptr_t)out_grad_rows | (u64)(grad_stride * size);
  if (out_grad_weights) addresses |= (u64)(uintptr_t)rows | (u64)(rows_stride * size);
  const int unit = unit_bytes(row_len * size, addresses);
  ScopedKernelTimer timer(ctx, KID_EXPERT_ROWS, stream);
  with_unit(dtype, unit, [&](auto value, auto bytes) {
    typedef decltype(value) T;
    constexpr int B = decltype(bytes)::value;
    const i64 units = row_len * size / B;
    const RowArgs a{tokens, num_rows, (int)per_token, 32, units, grad_stride * size / B, rows_stride * size / B,
                    place, Weights{weights, weights_dtype}, ctx_counters(ctx)};
    const int grid = (int)min((i64)kNumSMs * 32, (i64)grid_for(tokens * per_token * 32, kRowThreads));
    k_combine_grad<T, B><<<grid, kRowThreads, 0, stream>>>(a, (const Unit<T, B>*)grad, (const Unit<T, B>*)rows,
                                                           (Unit<T, B>*)out_grad_rows, out_grad_weights);
  });
  GSB_LAUNCH_OK();
  return GSB_OK;
}
