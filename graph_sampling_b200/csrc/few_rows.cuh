// Products by expert of little work: a step of a few tokens, a small minibatch.  No tensor cores: what counts is how soon the first weights
// are on their way and the last sum is written.
//
// A CTA takes four rows of an expert by 64 columns, or four rows by 64 columns of a weights' gradient.  The reduced index is spread over the
// lanes, whose sums meet by shuffles and, between warps, in shared memory, always in the same order.
#pragma once
#include <type_traits>

#include "group_plan.cuh"
#include "launch.cuh"
#include "row_values.cuh"

namespace gsb {

constexpr int kFewThreads = 256, kFewRows = 4, kFewColumns = 64, kFewDepth = 1024;

struct FewArgs {
  Groups groups;
  const void *rows, *other;  // of a product: its weights; of a gradient: the gradient's rows
  i64 rows_stride, other_stride, expert_stride;
  u32 k, n;
  const float *row_scales, *weight_scales;
};

// Up to eight neighbouring values as float.
template <class T, bool WIDE>
__device__ __forceinline__ void load_eight(const T* from, int valid, float (&f)[8]) {
  if (WIDE && valid >= 8) {
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int u = 0; u < 8 / N; ++u) {
      float g[N];
      load_unit((const Unit<T, 16>*)from + u).get(g);
#pragma unroll
      for (int q = 0; q < N; ++q) f[u * N + q] = g[q];
    }
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) f[q] = q < valid ? (float)from[q] : 0.f;
  }
}

// Sums of 4 rows by 8 columns a lane, over lanes 8 and 16 apart and over the warps: thread t gets that of row t / 64, column t % 64.
__device__ __forceinline__ float add_up(const float (&acc)[kFewRows][8], float (&room)[8][kFewRows][kFewColumns]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const bool upper = lane & 8, odd = lane & 16;
  float two[2][8], one[8];
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int q = 0; q < 8; ++q) two[r][q] = (upper ? acc[r + 2][q] : acc[r][q]) + __shfl_xor_sync(0xffffffffu, upper ? acc[r][q] : acc[r + 2][q], 8);
#pragma unroll
  for (int q = 0; q < 8; ++q) one[q] = (odd ? two[1][q] : two[0][q]) + __shfl_xor_sync(0xffffffffu, odd ? two[0][q] : two[1][q], 16);
  float* to = &room[warp][(upper ? 2 : 0) + (odd ? 1 : 0)][(lane & 7) * 8];
  __syncthreads();
  *(float4*)to = make_float4(one[0], one[1], one[2], one[3]);
  *(float4*)(to + 4) = make_float4(one[4], one[5], one[6], one[7]);
  __syncthreads();
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) sum += room[w][threadIdx.x / kFewColumns][threadIdx.x % kFewColumns];
  return sum;
}

template <class T>
__device__ __forceinline__ void clear_others(const Groups& g, const PlanTable& plan, u32 n, T* out) {
  const i64 step = (i64)gridDim.x * kFewThreads, at = (i64)blockIdx.x * kFewThreads + threadIdx.x;
  if (g.first == 0)
    for (i64 i = at; i < (i64)plan.begin[0] * n; i += step) out[i] = from_float<T>(0.f);
  if (g.first + g.experts == g.all)
    for (i64 i = (i64)plan.begin[g.experts] * n + at; i < (i64)g.num_rows * n; i += step) out[i] = from_float<T>(0.f);
}

// Weights whose rows are runs of memory: a lane takes 8 columns of every 32nd of them.
template <class T, bool WIDE>
__global__ void __launch_bounds__(kFewThreads) k_few_across(const FewArgs a, T* __restrict__ out) {
  __shared__ PlanTable plan;
  __shared__ __align__(16) float4 held[kFewDepth];  // the rows, by the reduced index
  __shared__ __align__(16) float room[8][kFewRows][kFewColumns];
  await_previous();
  const Groups& g = a.groups;
  make_plan<kFewThreads>(plan, g, kFewRows, 0);
  leave_end(plan, g);
  const u32 across = (a.n + kFewColumns - 1) / kFewColumns;
  const u64 tiles = (u64)plan.tile[g.experts] * across;
  const u32 part = threadIdx.x / 8, column = threadIdx.x % 8 * 8;
  for (u64 t = blockIdx.x; t < tiles; t += gridDim.x) {
    const u32 row_tile = (u32)(t / across), n0 = (u32)(t % across) * kFewColumns;
    const int e = expert_of_tile(plan, g.experts, row_tile);
    const u32 r0 = plan.begin[e] + (row_tile - plan.tile[e]) * kFewRows, valid = min((u32)kFewRows, plan.begin[e + 1] - r0);
    const T* weights = (const T*)a.other + (i64)(g.first + e) * a.expert_stride + n0 + column;
    const int columns = (int)a.n - (int)(n0 + column);
    const T* rows = (const T*)a.rows + (i64)r0 * a.rows_stride;
    float acc[kFewRows][8] = {};
    for (u32 k0 = 0; k0 < a.k; k0 += kFewDepth) {
      const u32 depth = min((u32)kFewDepth, a.k - k0);
      __syncthreads();
      for (u32 l = threadIdx.x; l < depth; l += kFewThreads) {
        float x[kFewRows];
#pragma unroll
        for (int r = 0; r < kFewRows; ++r) x[r] = (u32)r < valid ? (float)rows[r * a.rows_stride + k0 + l] : 0.f;
        held[l] = make_float4(x[0], x[1], x[2], x[3]);
      }
      __syncthreads();
#pragma unroll 8
      for (u32 l = part; l < depth; l += 32) {
        float w[8];
        load_eight<T, WIDE>(weights + (i64)(k0 + l) * a.other_stride, columns, w);
        const float4 x = held[l];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          acc[0][q] += x.x * w[q];
          acc[1][q] += x.y * w[q];
          acc[2][q] += x.z * w[q];
          acc[3][q] += x.w * w[q];
        }
      }
    }
    const float sum = add_up(acc, room);
    const u32 r = threadIdx.x / kFewColumns, c = n0 + threadIdx.x % kFewColumns;
    if (r < valid && c < a.n) out[(i64)(r0 + r) * a.n + c] = from_float<T>(sum);
  }
  clear_others(g, plan, a.n, out);
}

// Weights whose columns are runs of memory, in float types or (WHOLE) 8 bits: 8 lanes take 16 bytes each of two columns.
template <class T, class Out, bool WIDE>
__global__ void __launch_bounds__(kFewThreads) k_few_along(const FewArgs a, Out* __restrict__ out) {
  constexpr bool kWhole = std::is_same<T, signed char>::value;
  constexpr u32 kEach = kWhole ? 16 : 8;   // values of a lane and step
  typedef std::conditional_t<kWhole, int, float> Sum;
  typedef std::conditional_t<kWhole, int, float> Held;
  constexpr u32 kDepth = kWhole ? kFewDepth / 4 : kFewDepth;  // words of a row held
  __shared__ PlanTable plan;
  __shared__ __align__(16) Held held[kFewRows][kDepth];
  await_previous();
  const Groups& g = a.groups;
  make_plan<kFewThreads>(plan, g, kFewRows, 0);
  leave_end(plan, g);
  const u32 across = (a.n + kFewColumns - 1) / kFewColumns;
  const u64 tiles = (u64)plan.tile[g.experts] * across;
  const int lane = threadIdx.x & 31;
  const u32 part = threadIdx.x % 8 * kEach;
  for (u64 t = blockIdx.x; t < tiles; t += gridDim.x) {
    const u32 row_tile = (u32)(t / across), n0 = (u32)(t % across) * kFewColumns;
    const int e = expert_of_tile(plan, g.experts, row_tile);
    const u32 r0 = plan.begin[e] + (row_tile - plan.tile[e]) * kFewRows, valid = min((u32)kFewRows, plan.begin[e + 1] - r0);
    const u32 column[2] = {n0 + threadIdx.x / 8, n0 + threadIdx.x / 8 + 32};
    const T* rows = (const T*)a.rows + (i64)r0 * a.rows_stride;
    const T* weights = (const T*)a.other + (i64)(g.first + e) * a.expert_stride;
    Sum acc[2][kFewRows] = {};
    for (u32 k0 = 0; k0 < a.k; k0 += kFewDepth) {
      const u32 depth = min((u32)kFewDepth, a.k - k0);
      __syncthreads();
      if constexpr (kWhole) {
        for (u32 i = threadIdx.x; i < kFewRows * kDepth; i += kFewThreads) {
          const u32 r = i / kDepth, l = i % kDepth * 4;
          int w = 0;
          if (r < valid && l < depth) {
            const signed char* from = rows + r * a.rows_stride + k0 + l;
            if (l + 4 <= depth) w = *(const int*)from;
            else
              for (u32 q = 0; l + q < depth; ++q) w |= (from[q] & 255) << q * 8;
          }
          held[r][i % kDepth] = w;
        }
      } else {
        for (u32 i = threadIdx.x; i < kFewRows * kDepth; i += kFewThreads) {
          const u32 r = i / kDepth, l = i % kDepth;
          held[r][l] = r < valid && l < depth ? (float)rows[r * a.rows_stride + k0 + l] : 0.f;
        }
      }
      __syncthreads();
#pragma unroll 4
      for (u32 l = part; l < depth; l += 8 * kEach) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const T* from = weights + (i64)column[c] * a.other_stride + k0 + l;
          const int there = column[c] < a.n ? (int)(depth - l) : 0;
          if constexpr (kWhole) {
            int w[4] = {};
            if (there >= 16) {
              const int4 v = __ldg((const int4*)from);
              w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
            } else {
              for (int q = 0; q < there; ++q) w[q / 4] |= (from[q] & 255) << q % 4 * 8;
            }
#pragma unroll
            for (int r = 0; r < kFewRows; ++r) {
              const int4 x = *(const int4*)&held[r][l / 4];
              acc[c][r] = __dp4a(x.x, w[0], __dp4a(x.y, w[1], __dp4a(x.z, w[2], __dp4a(x.w, w[3], acc[c][r]))));
            }
          } else {
            float w[8];
            load_eight<T, WIDE>(from, there, w);
#pragma unroll
            for (int r = 0; r < kFewRows; ++r) {
              const float4 x = *(const float4*)&held[r][l], y = *(const float4*)&held[r][l + 4];
              acc[c][r] += x.x * w[0] + x.y * w[1] + x.z * w[2] + x.w * w[3] + (y.x * w[4] + y.y * w[5] + y.z * w[6] + y.w * w[7]);
            }
          }
        }
      }
    }
    // the 8 lanes of a column meet: each is left with one row of one column
    const bool second = lane & 4, upper = lane & 2, odd = lane & 1;
    Sum four[kFewRows], two[2];
#pragma unroll
    for (int r = 0; r < kFewRows; ++r) four[r] = (second ? acc[1][r] : acc[0][r]) + __shfl_xor_sync(0xffffffffu, second ? acc[0][r] : acc[1][r], 4);
#pragma unroll
    for (int r = 0; r < 2; ++r) two[r] = (upper ? four[r + 2] : four[r]) + __shfl_xor_sync(0xffffffffu, upper ? four[r] : four[r + 2], 2);
    const Sum sum = (odd ? two[1] : two[0]) + __shfl_xor_sync(0xffffffffu, odd ? two[0] : two[1], 1);
    const u32 r = (upper ? 2 : 0) + (odd ? 1 : 0), c = second ? column[1] : column[0];
    if (r < valid && c < a.n) {
      float v = (float)sum;
      if constexpr (kWhole) v = v * a.row_scales[r0 + r] * a.weight_scales[(i64)(g.first + e) * a.n + c];
      out[(i64)(r0 + r) * a.n + c] = from_float<Out>(v);
    }
  }
  clear_others(g, plan, a.n, out);
}

// The weights' gradient: a lane takes 8 columns of every 32nd row.
template <class T, bool WIDE>
__global__ void __launch_bounds__(kFewThreads) k_few_grad(const FewArgs a, T* __restrict__ out) {
  __shared__ PlanTable plan;
  __shared__ __align__(16) float room[8][kFewRows][kFewColumns];
  await_previous();
  const Groups& g = a.groups;
  make_plan<kFewThreads>(plan, g, 1, 0);
  leave_end(plan, g);
  const u32 across = (a.n + kFewColumns - 1) / kFewColumns, down = (a.k + kFewRows - 1) / kFewRows;
  const u64 tiles = (u64)g.experts * across * down;
  const u32 part = threadIdx.x / 8, column = threadIdx.x % 8 * 8;
  for (u64 t = blockIdx.x; t < tiles; t += gridDim.x) {
    const u32 e = (u32)(t / (across * down)), rest = (u32)(t - (u64)e * (across * down)), m0 = rest / across * kFewRows, n0 = rest % across * kFewColumns;
    const u32 valid = min((u32)kFewRows, a.k - m0);
    const int columns = (int)a.n - (int)(n0 + column);
    const T* rows = (const T*)a.rows + m0;
    const T* grad = (const T*)a.other + n0 + column;
    float acc[kFewRows][8] = {};
#pragma unroll 4
    for (u32 r = plan.begin[e] + part; r < plan.begin[e + 1]; r += 32) {
      float w[8];
      load_eight<T, WIDE>(grad + (i64)r * a.other_stride, columns, w);
#pragma unroll
      for (int i = 0; i < kFewRows; ++i) {
        const float x = (u32)i < valid ? (float)rows[(i64)r * a.rows_stride + i] : 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[i][q] += x * w[q];
      }
    }
    const float sum = add_up(acc, room);
    const u32 i = threadIdx.x / kFewColumns, c = n0 + threadIdx.x % kFewColumns;
    if (i < valid && c < a.n) out[((i64)(g.first + e) * a.k + m0 + i) * a.n + c] = from_float<T>(sum);
  }
}

}  // namespace gsb
