// Rows sorted by expert (or by node type) and back.
//
// Order: slot s = t * K + k of token t wants expert e(s), or none (-1).  Slots are sorted by expert, stably; those without one
// come last.  place[s] is the row of slot s in that order, ~row (negative) for a slot without an expert.
// Spread:  rows[place[t, k], :] = w[t, k] * x[t, :] (w = 1 without weights), zeros in the rows of slots without an expert.
// Combine: out[t, :] = sum over k of w[t, k] * rows[place[t, k], :], slots without an expert left out.
// Combine's gradient: spread of the output's gradient for the rows, and for w[t, k] the product <grad[t, :], rows[place[t, k], :]>.
// Spread's gradient is a combine.  Sums are in float, in the order of k; each result is rounded once.
//
// All are bound by DRAM: 500 000 rows of 1 KB spread in 151 us and combined in 158, 6.8 and 6.5 TB/s; 65 528 rows of 2 KB from and to
// 8 191 tokens spread in 25 us (6.0), combined in 28 (4.9, rows in no order), both with the weights' gradients in 50 (5.4).
#include <type_traits>

#include "key_sort.cuh"
#include "launch.cuh"
#include "row_values.cuh"
#include "scan.cuh"

namespace gsb {

constexpr int kRowThreads = 256;

enum { WEIGHTS_NONE, WEIGHTS_FLOAT, WEIGHTS_OF_ROWS };

// All counts are below 2^31: with 64-bit arithmetic there was more of that than of the rows' values (314 602 rows of 200 bytes spread in
// 45 us for 26).
struct RowArgs {
  u32 tokens, per_token, slots, num_rows;
  int lanes, units;                  // per group; per row
  i64 token_stride, row_stride;      // in units
  const i64* place;
  const void* weights;
  int weight_kind;
  i64* counters;
};

template <class T>
__device__ __forceinline__ float weight_at(const RowArgs& a, u32 slot) {
  if (a.weight_kind == WEIGHTS_NONE) return 1.f;
  if (a.weight_kind == WEIGHTS_FLOAT) return __ldg((const float*)a.weights + slot);
  float f[1];
  load_unit((const Unit<T, (int)sizeof(T)>*)a.weights + slot).get(f);
  return f[0];
}

// Row of a slot, or ~row for a slot without an expert.  kNowhere: out of range, which is recorded, unless it is the row of a
// slot without an expert that a caller's shorter array does not have.
constexpr int kNowhere = (int)0x80000000;
__device__ __forceinline__ int place_of(const RowArgs& a, u32 slot, bool report) {
  const i64 p = __ldg(a.place + slot);
  const u64 row = (u64)(p < 0 ? ~p : p);
  if (row < (u64)a.num_rows) return (int)p;
  if (report && (p >= 0 || row >= (u64)a.slots)) raise_error(a.counters, GSB_ERR_INDEX_RANGE, slot);
  return kNowhere;
}

// A group of lanes takes kTokens tokens at a time, a tile of their columns (blockIdx.y).
template <class T, int BYTES, int STEPS>
__global__ void __launch_bounds__(kRowThreads) k_spread_rows(const RowArgs a, const Unit<T, BYTES>* __restrict__ x,
                                                             Unit<T, BYTES>* __restrict__ rows) {
  constexpr int kTokens = rows_ahead(STEPS), N = Unit<T, BYTES>::N;
  await_previous();
  const int j = blockIdx.y * a.lanes * STEPS + (threadIdx.x & (a.lanes - 1));
  const u32 step = gridDim.x * (kRowThreads / a.lanes) * kTokens;
  bool in[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) in[s] = j + s * a.lanes < a.units;
  x += j;
  rows += j;
  for (u32 t = (blockIdx.x * kRowThreads + threadIdx.x) / a.lanes * kTokens; t < a.tokens; t += step) {
    Unit<T, BYTES> v[kTokens][STEPS];
#pragma unroll
    for (int r = 0; r < kTokens; ++r)
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        if (t + r < a.tokens && in[s]) v[r][s] = load_unit_once(x + (i64)(t + r) * a.token_stride + s * a.lanes);
    for (u32 k = 0; k < a.per_token; ++k) {
      int p[kTokens];
#pragma unroll
      for (int r = 0; r < kTokens; ++r) p[r] = t + r < a.tokens ? place_of(a, (t + r) * a.per_token + k, j == 0) : kNowhere;
#pragma unroll
      for (int r = 0; r < kTokens; ++r) {
        if (p[r] == kNowhere) continue;
        Unit<T, BYTES>* to = rows + (i64)(p[r] < 0 ? ~p[r] : p[r]) * a.units;
        if (a.weight_kind == WEIGHTS_NONE && p[r] >= 0) {
#pragma unroll
          for (int s = 0; s < STEPS; ++s)
            if (in[s]) store_unit_once(to + s * a.lanes, v[r][s]);
        } else {
          const float w = p[r] >= 0 ? weight_at<T>(a, (t + r) * a.per_token + k) : 0.f;
#pragma unroll
          for (int s = 0; s < STEPS; ++s) {
            Unit<T, BYTES> u;
            u.clear();
            if (p[r] >= 0) {
              float f[N];
              v[r][s].get(f);
#pragma unroll
              for (int q = 0; q < N; ++q) f[q] *= w;
              u.set(f);
            }
            if (in[s]) store_unit_once(to + s * a.lanes, u);
          }
        }
      }
    }
  }
}

// A group of lanes goes through the slots of its run of tokens, with the rows of the next kAhead slots on their way whatever
// token they belong to.
template <class T, int BYTES, int STEPS>
__global__ void __launch_bounds__(kRowThreads) k_combine_rows(const RowArgs a, u32 run, const Unit<T, BYTES>* __restrict__ rows,
                                                              Unit<T, BYTES>* __restrict__ out) {
  constexpr int N = Unit<T, BYTES>::N, kAhead = rows_ahead(STEPS);
  await_previous();
  const int j = blockIdx.y * a.lanes * STEPS + (threadIdx.x & (a.lanes - 1));
  const u32 first = (blockIdx.x * kRowThreads + threadIdx.x) / a.lanes * run;
  if (first >= a.tokens) return;
  const u32 begin = first * a.per_token, end = min(first + run, a.tokens) * a.per_token;
  bool in[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) in[s] = j + s * a.lanes < a.units;
  rows += j;
  out += (i64)first * a.units + j;
  float sum[STEPS][N] = {};
  u32 left = a.per_token;  // slots of the token that are still to come
  int p[kAhead];
  float w[kAhead];
  auto look = [&](u32 slot) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      p[u] = slot + u < end ? place_of(a, slot + u, j == 0) : -1;
      w[u] = p[u] >= 0 ? weight_at<T>(a, slot + u) : 0.f;
    }
  };
  look(begin);
  for (u32 slot = begin; slot < end; slot += kAhead) {
    Unit<T, BYTES> v[kAhead][STEPS];
    float factor[kAhead];
    bool there[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      there[u] = p[u] >= 0;
      factor[u] = w[u];
      if (there[u])
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
          if (in[s]) v[u][s] = load_unit_once(rows + p[u] * a.row_stride + s * a.lanes);
    }
    if (slot + kAhead < end) look(slot + kAhead);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (slot + u >= end) continue;
      if (there[u])
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
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
        if (in[s]) store_unit_once(out + s * a.lanes, r);
#pragma unroll
        for (int q = 0; q < N; ++q) sum[s][q] = 0.f;
      }
      out += a.units;
    }
  }
}

// A group of lanes takes a slot at a time (two cost warps: rows of 100 halves 34 us for 32).  The gradient of a token's output is
// read once per slot, from L1 or L2 after the first time.
template <class T, int BYTES, int STEPS, bool DOTS>
__global__ void __launch_bounds__(kRowThreads) k_combine_grad(const RowArgs a, const Unit<T, BYTES>* __restrict__ grad,
                                                              const Unit<T, BYTES>* __restrict__ rows,
                                                              Unit<T, BYTES>* __restrict__ grad_rows, void* grad_weights) {
  constexpr int N = Unit<T, BYTES>::N;
  await_previous();
  const int lane = threadIdx.x & (a.lanes - 1);
  const u32 step = gridDim.x * (kRowThreads / a.lanes);
  // all groups of a warp take part in the sums over lanes, also those that have run out of slots
  for (u32 base = (blockIdx.x * kRowThreads + (threadIdx.x & ~31u)) / a.lanes; base < a.slots; base += step) {
    const u32 slot = base + (threadIdx.x & 31) / a.lanes;
    const int p = slot < a.slots ? place_of(a, slot, lane == 0) : kNowhere;
    const float w = p >= 0 ? weight_at<T>(a, slot) : 0.f;
    const Unit<T, BYTES>* g_of = grad + (i64)(slot / a.per_token) * a.token_stride;
    const Unit<T, BYTES>* v_of = rows + (p >= 0 ? p : 0) * a.row_stride;
    Unit<T, BYTES>* to = grad_rows + (i64)(p < 0 ? ~p : p) * a.units;
    float dot = 0.f;
    for (int j = lane; j < a.units; j += a.lanes * STEPS) {
      Unit<T, BYTES> g[STEPS], v[STEPS];
      if (p >= 0)
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
          if (j + s * a.lanes < a.units) {
            if (DOTS) v[s] = load_unit_once(v_of + j + s * a.lanes);
            g[s] = load_unit(g_of + j + s * a.lanes);
          }
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        if (p == kNowhere || j + s * a.lanes >= a.units) continue;
        Unit<T, BYTES> u;
        u.clear();
        if (p >= 0) {
          float f[N], h[N];
          g[s].get(f);
          if (DOTS) {
            v[s].get(h);
#pragma unroll
            for (int q = 0; q < N; ++q) dot += f[q] * h[q];
          }
#pragma unroll
          for (int q = 0; q < N; ++q) f[q] *= w;
          u.set(f);
        }
        if (grad_rows) store_unit_once(to + j + s * a.lanes, u);
      }
    }
    if (!DOTS) continue;
    for (int o = a.lanes / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (lane != 0 || slot >= a.slots) continue;
    if (a.weight_kind == WEIGHTS_FLOAT) ((float*)grad_weights)[slot] = dot;
    else ((T*)grad_weights)[slot] = from_float<T>(dot);
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
  GSB_REQUIRE(aligned_to(8, (const char*)place) && (!weights || aligned_to(value_bytes(weights_dtype), (const char*)weights)),
              GSB_ERR_INVALID_ARGUMENT);
  return GSB_OK;
}

static RowArgs row_args(gsb_ctx* ctx, i64 tokens, i64 per_token, i64 num_rows, RowShape shape, i64 units, i64 token_stride,
                        i64 row_stride, const int64_t* place, const void* weights, int weights_dtype) {
  return RowArgs{(u32)tokens, (u32)per_token, (u32)(tokens * per_token), (u32)num_rows, shape.lanes, (int)units, token_stride,
                 row_stride, place, weights,
                 !weights ? WEIGHTS_NONE : weights_dtype == GSB_F32 ? WEIGHTS_FLOAT : WEIGHTS_OF_ROWS, ctx_counters(ctx)};
}

}  // namespace gsb

using namespace gsb;

extern "C" int64_t gsb_expert_order_workspace(int64_t n, int64_t num_experts) {
  if (n < 0 || n >= ((int64_t)1 << 31) || num_experts < 1 || num_experts > GSB_MAX_EXPERTS) return GSB_ERR_INVALID_ARGUMENT;
  return (int64_t)key_sort_bytes(n, num_experts);
}

static int order(gsb_ctx* ctx, void* stream_, const int64_t* experts, int64_t n, int64_t num_experts, int most_ctas,
                 int64_t* out_offsets, int64_t* out_source, int64_t* out_place, void* workspace, int64_t workspace_bytes) {
  GSB_ENTER(ctx);
  const int64_t need = gsb_expert_order_workspace(n, num_experts);
  GSB_REQUIRE(need >= 0 && out_offsets, GSB_ERR_INVALID_ARGUMENT);
  cudaStream_t stream = (cudaStream_t)stream_;
  if (n == 0) {
    GSB_CUDA_OK(cudaMemsetAsync(out_offsets, 0, (size_t)(num_experts + 1) * sizeof(int64_t), stream));
    return GSB_OK;
  }
  GSB_REQUIRE(experts && out_source && out_place && workspace, GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(aligned_to(8, experts, out_offsets, out_source, out_place) && aligned_to(256, (const char*)workspace),
              GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(workspace_bytes >= need, GSB_ERR_CAPACITY);
  SortCall call{KeySource{experts, n, num_experts, true, -1, ctx_counters(ctx)}, SORT_ORDER};
  call.offsets = out_offsets;
  call.order_source = out_source;
  call.place = out_place;
  ScopedKernelTimer timer(ctx, KID_KEY_SORT, stream);
  return key_sort(ctx, stream, call, workspace, nullptr, most_ctas);
}

extern "C" int gsb_expert_order(gsb_ctx* ctx, void* stream, const int64_t* experts, int64_t n, int64_t num_experts,
                                int64_t* out_offsets, int64_t* out_source, int64_t* out_place, void* workspace,
                                int64_t workspace_bytes) {
  return order(ctx, stream, experts, n, num_experts, kNumSMs, out_offsets, out_source, out_place, workspace, workspace_bytes);
}

extern "C" int gsb_selftest_expert_order(gsb_ctx* ctx, void* stream, const int64_t* experts, int64_t n, int64_t num_experts,
                                         int most_ctas, int64_t* out_offsets, int64_t* out_source, int64_t* out_place,
                                         void* workspace, int64_t workspace_bytes) {
  GSB_REQUIRE(most_ctas >= 1, GSB_ERR_INVALID_ARGUMENT);
  return order(ctx, stream, experts, n, num_experts, most_ctas, out_offsets, out_source, out_place, workspace, workspace_bytes);
}

extern "C" int gsb_expert_spread(gsb_ctx* ctx, void* stream_, const void* x, int dtype, int64_t tokens, int64_t per_token,
                                 int64_t row_len, int64_t x_stride, const int64_t* place, const void* weights,
                                 int weights_dtype, void* out_rows) {
  GSB_ENTER(ctx);
  const int st = check_rows(tokens, per_token, row_len, dtype, x_stride, place, weights, weights_dtype);
  if (st != GSB_OK) return st;
  if (tokens == 0) return GSB_OK;
  const int size = value_bytes(dtype);
  GSB_REQUIRE(x && out_rows && aligned_to(size, (const char*)x, (const char*)out_rows), GSB_ERR_INVALID_ARGUMENT);
  cudaStream_t stream = (cudaStream_t)stream_;
  const int unit = unit_bytes(row_len * size, (u64)(uintptr_t)x | (u64)(uintptr_t)out_rows | (u64)(x_stride * size));
  ScopedKernelTimer timer(ctx, KID_EXPERT_ROWS, stream);
  with_unit(dtype, unit, [&](auto value, auto bytes) {
    typedef decltype(value) T;
    constexpr int B = decltype(bytes)::value;
    const i64 units = row_len * size / B;
    const RowShape shape = row_shape(units, copy_steps(B), copy_wide(B));
    const RowArgs a = row_args(ctx, tokens, per_token, tokens * per_token, shape, units, x_stride * size / B, units, place, weights,
                               weights_dtype);
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
  const int size = value_bytes(dtype);
  GSB_REQUIRE((rows || num_rows == 0) && out && aligned_to(size, (const char*)rows, (const char*)out), GSB_ERR_INVALID_ARGUMENT);
  cudaStream_t stream = (cudaStream_t)stream_;
  const int unit = unit_bytes(row_len * size, (u64)(uintptr_t)rows | (u64)(uintptr_t)out | (u64)(rows_stride * size));
  ScopedKernelTimer timer(ctx, KID_EXPERT_ROWS, stream);
  with_unit(dtype, unit, [&](auto value, auto bytes) {
    typedef decltype(value) T;
    constexpr int B = decltype(bytes)::value;
    const i64 units = row_len * size / B;
    const RowShape shape = row_shape(units, copy_steps(B), copy_wide(B));
    const RowArgs a = row_args(ctx, tokens, per_token, num_rows, shape, units, units, rows_stride * size / B, place, weights,
                               weights_dtype);
    with_steps(shape.steps, [&](auto steps) {
      constexpr int S = decltype(steps)::value;
      // tokens per group of lanes: one while there are SMs without work
      const i64 tiles = grid_for(units, shape.lanes * S), run = tokens * tiles * shape.lanes / 32 / (kNumSMs * 128) + 1;
      const dim3 grid(grid_for((tokens + run - 1) / run * a.lanes, kRowThreads), (unsigned)tiles);
      launch_behind(stream, k_combine_rows<T, B, S>, grid, kRowThreads, a, (u32)run, (const Unit<T, B>*)rows,
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
  GSB_REQUIRE(aligned_to(size, (const char*)grad, (const char*)rows, (const char*)out_grad_rows) &&
                  (!out_grad_weights || aligned_to(value_bytes(weights_dtype), (const char*)out_grad_weights)),
              GSB_ERR_INVALID_ARGUMENT);
  u64 addresses = (u64)(uintptr_t)grad | (u64)(uintptr_t)out_grad_rows | (u64)(grad_stride * size);
  if (out_grad_weights) addresses |= (u64)(uintptr_t)rows | (u64)(rows_stride * size);
  const int unit = unit_bytes(row_len * size, addresses);
  ScopedKernelTimer timer(ctx, KID_EXPERT_ROWS, stream);
  with_unit(dtype, unit, [&](auto value, auto bytes) {
    typedef decltype(value) T;
    constexpr int B = decltype(bytes)::value;
    const i64 units = row_len * size / B;
    const RowShape shape = row_shape(units, copy_steps(B), copy_wide(B));
    const RowArgs a = row_args(ctx, tokens, per_token, num_rows, shape, units, grad_stride * size / B, rows_stride * size / B, place,
                               weights, weights_dtype);
    with_steps(shape.steps, [&](auto steps) {
      constexpr int S = decltype(steps)::value;
      const int grid = (int)min((i64)kNumSMs * 32, (i64)grid_for(tokens * per_token * a.lanes, kRowThreads));
      auto kernel = out_grad_weights ? k_combine_grad<T, B, S, true> : k_combine_grad<T, B, S, false>;
      launch_behind(stream, kernel, grid, kRowThreads, a, (const Unit<T, B>*)grad, (const Unit<T, B>*)rows,
                    (Unit<T, B>*)out_grad_rows, out_grad_weights);
    });
  });
  GSB_LAUNCH_OK();
  return GSB_OK;
}
