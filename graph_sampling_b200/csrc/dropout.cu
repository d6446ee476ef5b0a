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
  u32 limit;
  float scale;
};

__device__ __forceinline__ void drop(float (&f)[8], const U32x4& bits, u32 limit, float scale) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const u32 half = q & 1 ? bits.v[q / 2] >> 16 : bits.v[q / 2] & 0xffffu;
    f[q] = half >= limit ? f[q] * scale : 0.f;
  }
}

// A thread takes a block of 8 values.  WHOLE: a block's values are neighbours in memory and begin on 16-byte boundaries.
template <class T, bool WHOLE>
__global__ void __launch_bounds__(kDropThreads) k_dropout(const DropArgs a, const T* __restrict__ x, T* __restrict__ out) {
  await_previous();
  const u64 seed = a.seed_at ? *a.seed_at : a.seed;
  const i64 blocks = (a.count + 7) / 8, step = (i64)gridDim.x * kDropThreads;
  for (i64 b = (i64)blockIdx.x * kDropThreads + threadIdx.x; b < blocks; b += step) {
    const i64 i = b * 8;
    float f[8];
    const U32x4 bits = rand_block(seed, (u64)b, 0, STREAM_DROPOUT);
    if (WHOLE && i + 8 <= a.count) {
      const T* from = x + (a.stride == a.width ? i : i / a.width * a.stride + i % a.width);
      constexpr int kUnits = sizeof(T) / 2, N = 16 / sizeof(T);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        float g[N];
        load_unit_once((const Unit<T, 16>*)from + u).get(g);
#pragma unroll
        for (int q = 0; q < N; ++q) f[u * N + q] = g[q];
      }
      drop(f, bits, a.limit, a.scale);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        float g[N];
#pragma unroll
        for (int q = 0; q < N; ++q) g[q] = f[u * N + q];
        Unit<T, 16> w;
        w.set(g);
        store_unit_once((Unit<T, 16>*)(out + i) + u, w);
      }
    } else {
      i64 row = i / a.width, column = i - row * a.width;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        f[q] = i + q < a.count ? (float)x[row * a.stride + column] : 0.f;
        if (++column == a.width) column = 0, ++row;
      }
      drop(f, bits, a.limit, a.scale);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (i + q < a.count) out[i + q] = from_float<T>(f[q]);
    }
  }
}

}  // namespace gsb

using namespace gsb;

extern "C" int gsb_dropout(gsb_ctx* ctx, void* stream_, const void* x, int dtype, int64_t num_rows, int64_t row_len, int64_t x_stride, double p,
                           uint64_t seed, const uint64_t* seed_device, void* out) {
  GSB_ENTER(ctx);
  const int size = value_bytes(dtype);
  GSB_REQUIRE(num_rows >= 0 && row_len >= 0 && x_stride >= 0 && size != 0 && p >= 0.0 && p <= 1.0, GSB_ERR_INVALID_ARGUMENT);
  GSB_REQUIRE(row_len == 0 || num_rows <= ((int64_t)1 << 60) / row_len, GSB_ERR_INVALID_ARGUMENT);
  if (num_rows == 0 || row_len == 0) return GSB_OK;
  GSB_REQUIRE(x && out && aligned_to(size, (const char*)x, (const char*)out) && aligned_to(8, seed_device), GSB_ERR_INVALID_ARGUMENT);
  cudaStream_t stream = (cudaStream_t)stream_;
  DropArgs a{num_rows * row_len, row_len, num_rows == 1 ? row_len : x_stride, seed, (const u64*)seed_device, (u32)(p * 65536.0 + 0.5), 0.f};
  if (a.limit < 65536) a.scale = 65536.f / (float)(65536 - a.limit);
  const bool whole = aligned_to(16, (const char*)x, (const char*)out) && (a.stride == a.width || (a.width % 8 == 0 && a.stride * size % 16 == 0));
  const i64 blocks = (a.count + 7) / 8;
  const int grid = (int)min((i64)kNumSMs * 8, (i64)grid_for(blocks, kDropThreads));
  ScopedKernelTimer timer(ctx, KID_DROPOUT, stream);
  with_unit(dtype, size, [&](auto value, auto) {
    typedef decltype(value) T;
    if (whole) launch_behind(stream, k_dropout<T, true>, grid, kDropThreads, a, (const T*)x, (T*)out);
    else launch_behind(stream, k_dropout<T, false>, grid, kDropThreads, a, (const T*)x, (T*)out);
  });
  GSB_LAUNCH_OK();
  return GSB_OK;
}
