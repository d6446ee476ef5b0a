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
#include "launch.cuh"
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

// A group of lanes takes kTokens tokens at a time.
template <class T, int BYTES, int STEPS>
__global__ void __launch_bounds__(kRowThreads) k_spread_rows(const RowArgs a, const Unit<T, BYTES>* __restrict__ x,
                                                             Unit<T, BYTES>* __restrict__ rows) {
  constexpr int kTokens = rows_ahead(STEPS), N = Unit<T, BYTES>::N;
  await_previous();
  const int lane = threadIdx.x & (a.lanes - 1);
  const i64 j = (i64)blockIdx.y * a.lanes * STEPS + lane;
  const i64 step = (i64)gridDim.x * (kRowThreads / a.lanes) * kTokens;
  for (i64 t = ((i64)blockIdx.x * kRowThreads + threadIdx.x) / a.lanes * kTokens; t < a.tokens; t += step) {
    Unit<T, BYTES> v[kTokens][STEPS];
#pragma unroll
    for (int r = 0; r < kTokens; ++r)
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        if (t + r < a.tokens && j + s * a.lanes < a.units) v[r][s] = load_unit_once(x + (t + r) * a.token_stride + j + s * a.lanes);
    for (int k = 0; k < a.per_token; ++k) {
      i64 p[kTokens];
      float w[kTokens];
#pragma unroll
      for (int r = 0; r < kTokens; ++r) {
        const i64 slot = (t + r) * a.per_token + k;
        p[r] = t + r < a.tokens ? place_of(a, slot, j == 0) : kNowhere;
        w[r] = p[r] >= 0 && p[r] != kNowhere ? weight_of(a.weights, slot) : 0.f;
      }
#pragma unroll
      for (int r = 0; r < kTokens; ++r) {
        if (p[r] == kNowhere) continue;
        Unit<T, BYTES>* to = rows + (p[r] < 0 ? ~p[r] : p[r]) * a.units + j;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          Unit<T, BYTES> u = v[r][s];
          if (p[r] < 0) {
            u.clear();
          } else if (a.weights.p) {
            float f[N];
            u.get(f);
#pragma unroll
            for (int q = 0; q < N; ++q) f[q] *= w[r];
            u.set(f);
          }
          if (j + s * a.lanes < a.units) store_unit_once(to + s * a.lanes, u);
        }
      }
    }
  }
}

// A group of lanes goes through the slots of its run of tokens, with the rows of the next kAhead slots on their way whatever
// token they belong to.
template <class T, int BYTES, int STEPS>
__global__ void __launch_bounds__(kRowThreads) k_combine_rows(const RowArgs a, i64 run, const Unit<T, BYTES>* __restrict__ rows,
                                                              Unit<T, BYTES>* __restrict__ out) {
  constexpr int N = Unit<T, BYTES>::N, kAhead = rows_ahead(STEPS);
  await_previous();
  const int lane = threadIdx.x & (a.lanes - 1);
  const i64 j = (i64)blockIdx.y * a.lanes * STEPS + lane;
  const i64 first = ((i64)blockIdx.x * kRowThreads + threadIdx.x) / a.lanes * run;
  if (first >= a.tokens) return;
  const i64 begin = first * a.per_token, end = min(first + run, a.tokens) * a.per_token;
  Unit<T, BYTES>* to = out + first * a.units + j;
  float sum[STEPS][N] = {};
  int left = a.per_token;  // slots of the token that are still to come
  i64 p[kAhead];
  float w[kAhead];
  auto look = [&](i64 slot) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      p[u] = slot + u < end ? place_of(a, slot + u, j == 0) : -1;
      if (p[u] == kNowhere) p[u] = -1;
      w[u] = p[u] >= 0 ? weight_of(a.weights, slot + u) : 0.f;
    }
  };
  look(begin);
  for (i64 slot = begin; slot < end; slot += kAhead) {
    Unit<T, BYTES> v[kAhead][STEPS];
    float factor[kAhead];
    bool there[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      there[u] = p[u] >= 0;
      factor[u] = w[u];
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        if (there[u] && j + s * a.lanes < a.units) v[u][s] = load_unit_once(rows + p[u] * a.row_stride + j + s * a.lanes);
    }
    look(slot + kAhead);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (slot + u >= end) continue;
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        if (there[u] && j + s * a.lanes < a.units) {
          float f[N];
          v[u][s].get(f);
#pragma unroll
          for (int q = 0; q < N; ++q) sum[s][q] += f[q] * factor[u];
        }
      if (--left > 0) continue;
      left = a.per_token;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        Unit<T, BYTES> r;
        r.set(sum[s]);
        if (j + s * a.lanes < a.units) store_unit_once(to + s * a.lanes, r);
#pragma unroll
        for (int q = 0; q < N; ++q) sum[s][q] = 0.f;
      }
      to += a.units;
    }
  }
}

template <class W>
__device__ __forceinline__ void store_weight(void* p, i64 slot, float v) {
  ((W*)p)[slot] = from_float<W>(v);
}

// A group of lanes takes neighbouring slots at a time: one of rows in units of 16 bytes (two cost warps: 62 us for 58), two of
// narrower ones.  The gradient of a token's output is read once per slot, from L1 or L2 after the first time.
template <class T, int BYTES>
constexpr int grad_slots() { return BYTES == 16 ? 1 : 2; }

template <class T, int BYTES, int STEPS>
__global__ void __launch_bounds__(kRowThreads) k_combine_grad(const RowArgs a, const Unit<T, BYTES>* __restrict__ grad,
                                                              const Unit<T, BYTES>* __restrict__ rows,
                                                              Unit<T, BYTES>* __restrict__ grad_rows, void* grad_weights) {
  constexpr int N = Unit<T, BYTES>::N, kSlots = grad_slots<T, BYTES>();
  await_previous();
  const int lane = threadIdx.x & (a.lanes - 1);
  const i64 step = (i64)gridDim.x * (kRowThreads / a.lanes) * kSlots, slots = a.tokens * a.per_token;
  // all groups of a warp take part in the sums over lanes, also those that have run out of slots
  const i64 warp_first = ((i64)blockIdx.x * kRowThreads + (threadIdx.x & ~31)) / a.lanes * kSlots;
  for (i64 base = warp_first; base < slots; base += step) {
    const i64 slot = base + (threadIdx.x & 31) / a.lanes * kSlots;
    i64 p[kSlots], t[kSlots];
    bool there[kSlots];
    float w[kSlots], dot[kSlots] = {};
#pragma unroll
    for (int r = 0; r < kSlots; ++r) {
      p[r] = slot + r < slots ? place_of(a, slot + r, lane == 0) : kNowhere;
      t[r] = (u32)(slot + r) / (u32)a.per_token;
      there[r] = p[r] >= 0 && p[r] != kNowhere;
      w[r] = there[r] ? weight_of(a.weights, slot + r) : 0.f;
    }
    for (i64 j = lane; j < a.units; j += a.lanes * STEPS) {
      Unit<T, BYTES> g[kSlots][STEPS], v[kSlots][STEPS];
#pragma unroll
      for (int r = 0; r < kSlots; ++r)
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          if (!there[r] || j + s * a.lanes >= a.units) continue;
          if (grad_weights) v[r][s] = load_unit_once(rows + p[r] * a.row_stride + j + s * a.lanes);
          g[r][s] = load_unit(grad + t[r] * a.token_stride + j + s * a.lanes);
        }
#pragma unroll
      for (int r = 0; r < kSlots; ++r)
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          if (p[r] == kNowhere || j + s * a.lanes >= a.units) continue;
          Unit<T, BYTES> u;
          u.clear();
          if (there[r]) {
            float f[N], h[N];
            g[r][s].get(f);
            if (grad_weights) {
              v[r][s].get(h);
#pragma unroll
              for (int q = 0; q < N; ++q) dot[r] += f[q] * h[q];
            }
#pragma unroll
            for (int q = 0; q < N; ++q) f[q] *= w[r];
            u.set(f);
          }
          if (grad_rows) store_unit_once(grad_rows + (p[r] < 0 ? ~p[r] : p[r]) * a.units + j + s * a.lanes, u);
        }
    }
    if (!grad_weights) continue;
#pragma unroll
    for (int r = 0; r < kSlots; ++r) {
      for (int o = a.lanes / 2; o > 0; o >>= 1) dot[r] += __shfl_xor_sync(0xffffffffu, dot[r], o);
      if (lane != 0 || slot + r >= slots) continue;
      if (a.weights.dtype == GSB_F32) store_weight<float>(grad_weights, slot + r, dot[r]);
      else if (a.weights.dtype == GSB_F16) store_weight<__half>(grad_weights, slot + r, dot[r]);
      else store_weight<__nv_bfloat16>(grad_weights, slot + r, dot[r]);
    }
  }
}

static int check_rows(i64 tokens, i64 per_token, i64 row_len, int dtype, i64 stride, const void* place, const void* weights,
                      int weights_dtype) {
  GSB_REQUIRE(tokens >= 0 && per_token >= 1 && tokens < ((i64)1 << 31) && per_token < ((i64)1 << 31) &&
                  tokens * per_token < ((i64)1 << 31) && row_len >= 1 && row_len <= GSB_MAX_ROW_LEN &&
                  stride >= 0 && value_bytes(dtype) != 0,
              GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(tokens == 0 || place, GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(!weights || weights_dtype == dtype || weights_dtype == GSB_F32, GSB_ERR_INVALID_ARGUMENT);
  return GSB_OK;
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
    const RowShape shape = row_shape(units, copy_steps(B));
    const RowArgs a{tokens, tokens * per_token, (int)per_token, shape.lanes, units, x_stride * size / B, units,
                    place, Weights{weights, weights_dtype}, ctx_counters(ctx)};
    with_steps(shape.steps, [&](auto steps) {
      constexpr int S = decltype(steps)::value, kTokens = rows_ahead(S);
      const dim3 grid((unsigned)min((i64)kNumSMs * 32, (i64)grid_for((tokens + kTokens - 1) / kTokens * a.lanes, kRowThreads)),
                      grid_for(units, shape.lanes * S));
      launch_behind(stream, k_spread_rows<T, B, S>, grid, kRowThreads, a, (const Unit<T, B>*)x,
                    (Unit<T, B>*)out_rows);
    });
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
    const RowShape shape = row_shape(units, copy_steps(B));
    const RowArgs a{tokens, num_rows, (int)per_token, shape.lanes, units, units, rows_stride * size / B,
                    place, Weights{weights, weights_dtype}, ctx_counters(ctx)};
    with_steps(shape.steps, [&](auto steps) {
      constexpr int S = decltype(steps)::value;
      // tokens per group of lanes: one while there are SMs without work
      const i64 tiles = grid_for(units, shape.lanes * S), run = tokens * tiles * shape.lanes / 32 / (kNumSMs * 128) + 1;
      const dim3 grid(grid_for((tokens + run - 1) / run * a.lanes, kRowThreads), (unsigned)tiles);
      launch_behind(stream, k_combine_rows<T, B, S>, grid, kRowThreads, a, run, (const Unit<T, B>*)rows,
                    (Unit<T, B>*)out);
    });
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
    const RowShape shape = row_shape(units, copy_steps(B));
    const RowArgs a{tokens, num_rows, (int)per_token, shape.lanes, units, grad_stride * size / B, rows_stride * size / B,
                    place, Weights{weights, weights_dtype}, ctx_counters(ctx)};
    with_steps(shape.steps, [&](auto steps) {
      constexpr int S = decltype(steps)::value, kSlots = grad_slots<T, B>();
      const int grid = (int)min((i64)kNumSMs * 32, (i64)grid_for((tokens * per_token + kSlots - 1) / kSlots * a.lanes, kRowThreads));
      launch_behind(stream, k_combine_grad<T, B, S>, grid, kRowThreads, a, (const Unit<T, B>*)grad,
                    (const Unit<T, B>*)rows, (Unit<T, B>*)out_grad_rows, out_grad_weights);
    });
  });
  GSB_LAUNCH_OK();
  return GSB_OK;
}
