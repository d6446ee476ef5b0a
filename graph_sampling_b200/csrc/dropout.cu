// Dropout whose mask is never stored: the backward pass makes it again.
//
// Value i, in the row-major order of the tensor, belongs to the 16 bits number i % 8 of block i / 8 of the counter-based generator under
// the call's seed.  It is dropped (0, whatever it was) where they are below limit = p * 65 536, rounded, and multiplied with
// 65 536 / (65 536 - limit) where they are not: the probability is a multiple of 2^-16, and the mean is kept exactly for it.
#include "launch.cuh"
#include "philox.cuh"
#include "row_values.cuh"

namespace gsb {

constexpr int kDropThreads = 256;

struct DropArgs {
  i64 count, width, stride;  // values; of a row; from a row's start to the next
  u64 seed;
  const u64* seed_at;        // where the seed is, on the device (null: `seed`)
  u32 limit;                 // in the upper half: below 2^16
  float scale;
};

// Bits in the upper half of a word are compared as the whole word: what is below them does not decide.
__device__ __forceinline__ void drop(float (&f)[8], const U32x4& bits, u32 limit, float scale) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const u32 half = q & 1 ? bits.v[q / 2] : bits.v[q / 2] << 16;
    f[q] = half >= limit ? f[q] * scale : 0.f;
  }
}

// A thread takes kBlocks blocks of 8 values, and no more: a million rows of 602 bf16 take 360 us (6.7 TB/s), with two blocks 380, with a
// grid that fills the GPU once and goes on in steps 449.
constexpr int kBlocks = 4;

// A block's values are neighbours in memory and begin on 16-byte boundaries, in rows (ROWS) or in one run.
template <class T, bool ROWS>
__global__ void __launch_bounds__(kDropThreads) k_dropout(const DropArgs a, const T* __restrict__ x, T* __restrict__ out) {
  constexpr int kUnits = sizeof(T) / 2, N = 16 / sizeof(T);
  typedef Unit<T, 16> U;
  await_previous();
  const u64 seed = a.seed_at ? *a.seed_at : a.seed;
  const i64 blocks = a.count / 8, b0 = (i64)blockIdx.x * (kDropThreads * kBlocks) + threadIdx.x;
  U v[kBlocks][kUnits];
#pragma unroll
  for (int k = 0; k < kBlocks; ++k) {
    const i64 b = b0 + k * kDropThreads;
    if (b < blocks) {
      const T* from = x + (ROWS ? b * 8 / a.width * a.stride + b * 8 % a.width : b * 8);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) v[k][u] = load_unit_once((const U*)from + u);
    }
  }
#pragma unroll
  for (int k = 0; k < kBlocks; ++k) {
    const i64 b = b0 + k * kDropThreads;
    if (b >= blocks) continue;
    const U32x4 bits = rand_block(seed, (u64)b, 0, STREAM_DROPOUT);
    float f[8];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      float g[N];
      v[k][u].get(g);
#pragma unroll
      for (int q = 0; q < N; ++q) f[u * N + q] = g[q];
    }
    drop(f, bits, a.limit, a.scale);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      float g[N];
#pragma unroll
      for (int q = 0; q < N; ++q) g[q] = f[u * N + q];
      U w;
      w.set(g);
      store_unit_once((U*)(out + b * 8) + u, w);
    }
  }
}

// Any addresses and distances, from block `first` on.
template <class T>
__global__ void __launch_bounds__(kDropThreads) k_dropout_any(const DropArgs a, i64 first, const T* __restrict__ x, T* __restrict__ out) {
  await_previous();
  const u64 seed = a.seed_at ? *a.seed_at : a.seed;
  const i64 blocks = (a.count + 7) / 8, step = (i64)gridDim.x * kDropThreads;
  for (i64 b = first + (i64)blockIdx.x * kDropThreads + threadIdx.x; b < blocks; b += step) {
    const i64 i = b * 8;
    float f[8];
    i64 row = i / a.width, column = i - row * a.width;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      f[q] = i + q < a.count ? (float)x[row * a.stride + column] : 0.f;
      if (++column == a.width) column = 0, ++row;
    }
    drop(f, rand_block(seed, (u64)b, 0, STREAM_DROPOUT), a.limit, a.scale);
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (i + q < a.count) out[i + q] = from_float<T>(f[q]);
  }
}

}  // namespace gsb

using namespace gsb;

extern "C" int gsb_dropout(gsb_ctx* ctx, void* stream_, const void* x, int dtype, int64_t num_rows, int64_t row_len, int64_t x_stride, double p,
                           uint64_t seed, const uint64_t* seed_device, void* out) {
  GSB_ENTER(ctx);
  const int size = value_bytes(dtype);
  GSB_REQUIRE(num_rows >= 0 && row_len >= 0 && x_stride >= 0 && size != 0 && p >= 0.0 && p <= 1.0, GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(row_len == 0 || num_rows <= ((int64_t)1 << 43) / row_len, GSB_ERR_INVALID_ARGUMENT);
  if (num_rows == 0 || row_len == 0) return GSB_OK;
  GSB_REQUIRE(x && out && aligned_to(size, (const char*)x, (const char*)out) && aligned_to(8, seed_device), GSB_ERR_INVALID_ARGUMENT);
  cudaStream_t stream = (cudaStream_t)stream_;
  const u32 limit = (u32)(p * 65536.0 + 0.5);
  const i64 count = num_rows * row_len;
  if (limit == 65536) {
    GSB_CUDA_OK(cudaMemsetAsync(out, 0, (size_t)(count * size), stream));
    return GSB_OK;
  }
  const DropArgs a{count, row_len, num_rows == 1 ? row_len : x_stride, seed, (const u64*)seed_device, limit << 16, 65536.f / (float)(65536 - limit)};
  const bool run = a.stride == a.width;
  const bool whole = aligned_to(16, (const char*)x, (const char*)out) && (run || (a.width % 8 == 0 && a.stride * size % 16 == 0));
  const i64 first = whole ? count / 8 : 0, rest = (count + 7) / 8 - first;
  ScopedKernelTimer timer(ctx, KID_DROPOUT, stream);
  with_unit(dtype, size, [&](auto value, auto) {
    typedef decltype(value) T;
    if (first > 0) {
      const int grid = grid_for(first, kDropThreads * kBlocks);
      if (run) launch_behind(stream, k_dropout<T, false>, grid, kDropThreads, a, (const T*)x, (T*)out);
      else launch_behind(stream, k_dropout<T, true>, grid, kDropThreads, a, (const T*)x, (T*)out);
    }
    if (rest > 0)
      launch_behind(stream, k_dropout_any<T>, (int)min((i64)kNumSMs * 8, (i64)grid_for(rest, kDropThreads)), kDropThreads, a, first, (const T*)x, (T*)out);
  });
  GSB_LAUNCH_OK();
  return GSB_OK;
}
