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

// BYTES of neighbouring memory by one access.
template <int BYTES>
__device__ __forceinline__ void load_words(const void* from, u32 (&w)[BYTES / 4]) {
  if constexpr (BYTES == 32) {
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(from) : "memory");
  } else {
    const uint4 v = __ldcs((const uint4*)from);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
}
template <int BYTES>
__device__ __forceinline__ void store_words(void* to, const u32 (&w)[BYTES / 4]) {
  if constexpr (BYTES == 32) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 :: "l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
  } else {
    __stcs((uint4*)to, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// A piece is what a thread reads at a time: 32 bytes by one access where addresses allow it, else a block of 8 values, 16 bytes an access.
template <class T, int BYTES>
struct Piece {
  static constexpr int kValues = (BYTES < 8 * (int)sizeof(T) ? 8 * (int)sizeof(T) : BYTES) / (int)sizeof(T), kBlocks = kValues / 8;
};

// A thread takes kDropBlocks blocks, and no more: a million rows of 602 bf16 take 347 us by 32 bytes an access (6.9 TB/s) and 369 by 16; by
// 16, with two blocks 380, with a grid that fills the GPU once and goes on in steps 449.
constexpr int kDropBlocks = 4;

// Pieces do not cross the ends of rows (ROWS), or there is one run.
template <class T, int BYTES, bool ROWS>
__global__ void __launch_bounds__(kDropThreads) k_dropout(const DropArgs a, const T* __restrict__ x, T* __restrict__ out) {
  typedef Piece<T, BYTES> P;
  typedef Unit<T, 16> U;
  constexpr int N = 16 / sizeof(T), kUnits = 8 / N, kPieces = kDropBlocks / P::kBlocks, kAccesses = P::kValues * (int)sizeof(T) / BYTES;
  await_previous();
  const u64 seed = a.seed_at ? *a.seed_at : a.seed;
  const i64 pieces = a.count / P::kValues, p0 = (i64)blockIdx.x * (kDropThreads * kPieces) + threadIdx.x;
  u32 w[kPieces][kAccesses][BYTES / 4];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const i64 i = (p0 + k * kDropThreads) * P::kValues;
    if (p0 + k * kDropThreads < pieces) {
      const T* from = x + (ROWS ? i / a.width * a.stride + i % a.width : i);
#pragma unroll
      for (int j = 0; j < kAccesses; ++j) load_words<BYTES>((const char*)from + j * BYTES, w[k][j]);
    }
  }
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const i64 p = p0 + k * kDropThreads;
    if (p >= pieces) continue;
#pragma unroll
    for (int block = 0; block < P::kBlocks; ++block) {
      const U32x4 bits = rand_block(seed, (u64)(p * P::kBlocks + block), 0, STREAM_DROPOUT);
      float f[8];
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int j = (block * kUnits + u) * 4;  // the unit's first word
        float g[N];
        U{make_uint4(w[k][j * 4 / BYTES][j % (BYTES / 4)], w[k][j * 4 / BYTES][(j + 1) % (BYTES / 4)], w[k][j * 4 / BYTES][(j + 2) % (BYTES / 4)],
                     w[k][j * 4 / BYTES][(j + 3) % (BYTES / 4)])}
            .get(g);
#pragma unroll
        for (int q = 0; q < N; ++q) f[u * N + q] = g[q];
      }
      drop(f, bits, a.limit, a.scale);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int j = (block * kUnits + u) * 4;
        float g[N];
#pragma unroll
        for (int q = 0; q < N; ++q) g[q] = f[u * N + q];
        U unit;
        unit.set(g);
        u32(&to)[BYTES / 4] = w[k][j * 4 / BYTES];
        to[j % (BYTES / 4)] = unit.w.x, to[(j + 1) % (BYTES / 4)] = unit.w.y, to[(j + 2) % (BYTES / 4)] = unit.w.z, to[(j + 3) % (BYTES / 4)] = unit.w.w;
      }
    }
#pragma unroll
    for (int j = 0; j < kAccesses; ++j) store_words<BYTES>((char*)(out + p * P::kValues) + j * BYTES, w[k][j]);
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
  // what one access can take of every row, or of the run; 0: a value
  auto divides = [&](int bytes) {
    const int values = max(8, bytes / size);
    return aligned_to(bytes, (const char*)x, (const char*)out) && (run || (a.width % values == 0 && a.stride * size % bytes == 0)) ? values : 0;
  };
  const int wide = divides(32), values = wide ? wide : divides(16);
  const i64 pieces = values ? count / values : 0, first = pieces * (values / 8), rest = (count + 7) / 8 - first;
  ScopedKernelTimer timer(ctx, KID_DROPOUT, stream);
  with_unit(dtype, size, [&](auto value, auto) {
    typedef decltype(value) T;
    if (pieces > 0) {
      auto* const kernel = wide ? (run ? k_dropout<T, 32, false> : k_dropout<T, 32, true>) : (run ? k_dropout<T, 16, false> : k_dropout<T, 16, true>);
      launch_behind(stream, kernel, grid_for(pieces, kDropThreads * kDropBlocks * 8 / values), kDropThreads, a, (const T*)x, (T*)out);
    }
    if (rest > 0)
      launch_behind(stream, k_dropout_any<T>, (int)min((i64)kNumSMs * 8, (i64)grid_for(rest, kDropThreads)), kDropThreads, a, first, (const T*)x, (T*)out);
  });
  GSB_LAUNCH_OK();
  return GSB_OK;
}
