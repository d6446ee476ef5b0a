// Rows in 8 bits with a scale each: scale[r] = max |x[r, :]| / 127, values[r, :] = x[r, :] / scale[r], rounded to the nearest whole
// number, ties to even.  Divisions are those of IEEE float, so the same rows give the same values wherever that is done.  A row of
// zeros has the scale 0; one that holds an infinity or NaN has a NaN for its scale, and zeros for its values.
#include "launch.cuh"
#include "row_values.cuh"

namespace gsb {

constexpr int kQuantThreads = 256;

// Two floats as one register pair.
__device__ __forceinline__ u64 pair_of(float a, float b) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 of_pair(u64 p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ u64 fma_pair(u64 a, u64 b, u64 c) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ u64 add_pair(u64 a, u64 b) {
  u64 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// f / scale to the nearest whole numbers, each in the low byte of q.  f * (1 / scale) is within 127 * 2^-22 of the quotient, so the whole number
// next to it is the right one unless it is as close to one half; then, and where the reciprocal is none, the quotient decides.
__device__ __forceinline__ int by_quotient(float v, float scale) { return scale > 0.f ? min(127, max(-127, __float2int_rn(__fdiv_rn(v, scale)))) : 0; }
template <int N>
__device__ __forceinline__ void quantized(const float (&f)[N], float scale, float inverse, int (&q)[N]) {
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it leaves the whole number in the low bits
  float off[N], worst = inverse > 0.f ? 0.f : 1.f;
  if constexpr (N > 1) {  // two values an instruction
    const u64 times = pair_of(inverse, inverse), minus = pair_of(-inverse, -inverse);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const u64 v = pair_of(f[i], f[i + 1]), near = fma_pair(v, times, pair_of(kRound, kRound));
      const float2 whole = of_pair(near), apart = of_pair(fma_pair(v, minus, add_pair(near, pair_of(-kRound, -kRound))));
      off[i] = apart.x, off[i + 1] = apart.y;
      q[i] = __float_as_int(whole.x), q[i + 1] = __float_as_int(whole.y);
      worst = fmaxf(fmaxf(worst, fabsf(off[i])), fabsf(off[i + 1]));
    }
  } else {
    const float near = __fmaf_rn(f[0], inverse, kRound);
    off[0] = __fmaf_rn(f[0], inverse, -(near - kRound));
    worst = fmaxf(worst, fabsf(off[0]));
    q[0] = __float_as_int(near);
  }
  if (worst < 0.4999f) return;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (!(fabsf(off[i]) < 0.4999f)) q[i] = by_quotient(f[i], scale);
}

// The largest size of a unit's values: of 16-bit ones two at a time, as the whole numbers that their bits are (infinities and NaN are above all
// others).
template <class T, int BYTES>
struct Largest {
  static constexpr bool kWords = sizeof(T) == 2 && BYTES >= 4;
  u32 bits = 0;
  __device__ __forceinline__ void look(const Unit<T, BYTES>& unit) {
    if constexpr (kWords) {
      u32 w[BYTES / 4];
      if constexpr (BYTES == 4) w[0] = unit.w;
      else if constexpr (BYTES == 8) w[0] = unit.w.x, w[1] = unit.w.y;
      else w[0] = unit.w.x, w[1] = unit.w.y, w[2] = unit.w.z, w[3] = unit.w.w;
#pragma unroll
      for (int i = 0; i < BYTES / 4; ++i) bits = __vmaxu2(bits, w[i] & 0x7fff7fffu);
    } else {
      float f[Unit<T, BYTES>::N];
      unit.get(f);
#pragma unroll
      for (int i = 0; i < Unit<T, BYTES>::N; ++i) bits = max(bits, __float_as_uint(f[i]) & 0x7fffffffu);
    }
  }
  __device__ __forceinline__ void look_value(unsigned short value) { bits = __vmaxu2(bits, value & 0x7fffu); }  // of 16 bits
  // of all lanes, or of `lanes` neighbouring ones; NaN where one is an infinity or NaN
  __device__ __forceinline__ float of_warp() const { return checked(__reduce_max_sync(0xffffffffu, as_float())); }
  __device__ __forceinline__ float of_lanes(int lanes) const {
    u32 most = as_float();
    for (int o = lanes / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    return checked(most);
  }

 private:
  __device__ __forceinline__ u32 as_float() const {
    if constexpr (kWords) {
      const u32 half = max(bits & 0xffffu, bits >> 16);
      return __float_as_uint(std::is_same<T, __half>::value ? __half2float(__ushort_as_half((unsigned short)half)) : __uint_as_float(half << 16)) & 0x7fffffffu;
    } else {
      return bits;
    }
  }
  static __device__ __forceinline__ float checked(u32 most) { return __uint_as_float(most >= 0x7f800000u ? 0x7fffffffu : most); }
};

__device__ __forceinline__ float inverse_of(float scale) { return scale > 1e-30f ? __fdiv_rn(1.f, scale) : __int_as_float(0x7fffffff); }
// PACKED: the N values of a unit are written as one word.
template <bool PACKED, class T, int BYTES>
__device__ __forceinline__ void put(const Unit<T, BYTES>& unit, int8_t* to, float scale, float inverse) {
  constexpr int N = Unit<T, BYTES>::N;
  float f[N];
  int q[N];
  unit.get(f);
  quantized(f, scale, inverse, q);
  if constexpr (PACKED && N == 2) {
    __stcs((unsigned short*)to, (unsigned short)__byte_perm(q[0], q[1], 0x0040));
  } else if constexpr (PACKED) {
    u32 w[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
      w[i] = __byte_perm(__byte_perm(q[4 * i], q[4 * i + 1], 0x0040), __byte_perm(q[4 * i + 2], q[4 * i + 3], 0x0040), 0x5410);
    if constexpr (N == 8) __stcs((uint2*)to, make_uint2(w[0], w[1]));
    else __stcs((u32*)to, w[0]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) to[i] = (int8_t)q[i];
  }
}

// Short rows: `lanes` neighbouring lanes (a power of two) take a row, kSteps units each, and kRows rows at a time.
constexpr int kShortRows = 4, kShortSteps = 2;
template <class T, int BYTES, bool PACKED>
__global__ void __launch_bounds__(kQuantThreads) k_quantize_short(const Unit<T, BYTES>* __restrict__ x, i64 x_stride, int units, int lanes, u32 num_rows,
                                                                  int8_t* __restrict__ values, i64 values_stride, float* __restrict__ scales) {
  constexpr int N = Unit<T, BYTES>::N;
  await_previous();
  const int lane = threadIdx.x & (lanes - 1);
  const u32 groups = kQuantThreads / lanes, first = blockIdx.x * groups * kShortRows + threadIdx.x / lanes;
  Unit<T, BYTES> v[kShortRows][kShortSteps];
#pragma unroll
  for (int r = 0; r < kShortRows; ++r)
#pragma unroll
    for (int s = 0; s < kShortSteps; ++s) {
      v[r][s].clear();
      if (first + r * groups < num_rows && lane + s * lanes < units) v[r][s] = load_unit_once(x + (i64)(first + r * groups) * x_stride + lane + s * lanes);
    }
#pragma unroll
  for (int r = 0; r < kShortRows; ++r) {
    const u32 row = first + r * groups;
    Largest<T, BYTES> largest;
#pragma unroll
    for (int s = 0; s < kShortSteps; ++s) largest.look(v[r][s]);
    const float scale = __fdiv_rn(largest.of_lanes(lanes), 127.f), inverse = inverse_of(scale);
    if (row >= num_rows) continue;
    if (lane == 0) scales[row] = scale;
#pragma unroll
    for (int s = 0; s < kShortSteps; ++s)
      if (lane + s * lanes < units) put<PACKED>(v[r][s], values + (i64)row * values_stride + (i64)(lane + s * lanes) * N, scale, inverse);
  }
}

// A warp takes a row.  Its first kHeld units stay in shared memory between the search for the largest value and the division (in registers
// the unrolled divisions were more code than the instruction cache holds: 65 536 rows of 2 048 bf16 took 184 us).  They take 71 (5.7 TB/s), 200 000
// rows of 608 take 90: the instructions of a row bound it, so one of up to 128 units is asked for by 4 to a lane at once, not 8 (90 and 101 us).
constexpr int kHeld = 256;
// Counted in warps: threads of 2^27 rows are more than 32 bits hold.
__device__ __forceinline__ u32 row_of_warp() { return blockIdx.x * (kQuantThreads / 32) + threadIdx.x / 32; }
template <class T, int BYTES, bool PACKED, int kAhead>
__global__ void __launch_bounds__(kQuantThreads) k_quantize_rows(const Unit<T, BYTES>* __restrict__ x, i64 x_stride, int units, u32 num_rows,
                                                                 int8_t* __restrict__ values, i64 values_stride, float* __restrict__ scales) {
  constexpr int N = Unit<T, BYTES>::N;
  typedef Unit<T, BYTES> U;
  typedef typename WordOf<BYTES>::type Word;
  __shared__ Word room[kQuantThreads / 32][kHeld];
  await_previous();
  const int lane = threadIdx.x & 31;
  Word* const held = room[threadIdx.x / 32];
  for (u32 r = row_of_warp(); r < num_rows; r += gridDim.x * (kQuantThreads / 32)) {
    const U* row = x + (i64)r * x_stride;
    Largest<T, BYTES> largest;
    for (int j0 = lane; j0 < units; j0 += 32 * kAhead) {
      U v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        v[u].clear();
        if (j0 + u * 32 < units) v[u] = load_unit_once(row + j0 + u * 32);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        largest.look(v[u]);
        if (j0 + u * 32 < kHeld) held[j0 + u * 32] = v[u].w;
      }
    }
    const float scale = __fdiv_rn(largest.of_warp(), 127.f);
    const float inverse = inverse_of(scale);
    if (lane == 0) scales[r] = scale;
    int8_t* const to_row = values + (i64)r * values_stride;
#pragma unroll 2
    for (int j = lane; j < units; j += 32) {
      U unit;
      if (j < kHeld) unit.w = held[j];
      else unit = load_unit(row + j);
      put<PACKED>(unit, to_row + (i64)j * N, scale, inverse);
    }
  }
}

// Long rows of 16-bit values that do not all begin on 16-byte boundaries: a warp brings a row's whole 16-byte lines to shared memory, its ends by
// values, and reads four values at a time there, from wherever they begin: 400 000 rows of 601 bf16 take 205 us, 100 000 of 1 319 take 97 (4.1
// TB/s); value by value they took 352 and 230.  What bounds it is the number of instructions.
constexpr int kShiftedRoom = 384;  // lines of a warp
template <class T>
__global__ void __launch_bounds__(kQuantThreads, 6) k_quantize_shifted(const T* __restrict__ x, i64 x_stride, int row_len, u32 num_rows,
                                                                    int8_t* __restrict__ values, i64 values_stride, float* __restrict__ scales, int room) {
  constexpr int kAhead = 4;
  extern __shared__ uint4 rooms[];
  await_previous();
  const int lane = threadIdx.x & 31;
  uint4* const held = rooms + threadIdx.x / 32 * room;
  for (u32 r = row_of_warp(); r < num_rows; r += gridDim.x * (kQuantThreads / 32)) {
    const T* row = x + (i64)r * x_stride;
    const int lead = (int)((u64)(uintptr_t)row & 15) / 2, end = lead + row_len, first = lead ? 1 : 0, last = end / 8;
    const Unit<T, 16>* lines = (const Unit<T, 16>*)(row - lead);
    Largest<T, 16> largest;
    const int at_end = lane < 8 ? lane : last * 8 + lane - 8;
    const bool ends = lane < 8 ? lead > 0 && lane >= lead : lane < 16 && at_end < end;
    unsigned short value = 0;
    if (ends) value = __ldcs((const unsigned short*)lines + at_end);
    for (int j0 = first + lane; j0 < last; j0 += 32 * kAhead) {
      Unit<T, 16> v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        v[u].clear();
        if (j0 + u * 32 < last) v[u] = load_unit_once(lines + j0 + u * 32);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        largest.look(v[u]);
        if (j0 + u * 32 < last) held[j0 + u * 32] = v[u].w;
      }
    }
    largest.look_value(value);
    if (ends) ((unsigned short*)held)[at_end] = value;
    const float scale = __fdiv_rn(largest.of_warp(), 127.f);
    const float inverse = inverse_of(scale);
    if (lane == 0) scales[r] = scale;
    __syncwarp();
    int8_t* const to = values + (i64)r * values_stride;
    const int skip = min(row_len, (int)(-(u64)(uintptr_t)to & 3)), words = (row_len - skip) / 4;
    const u32* const from = (const u32*)held + (lead + skip) / 2;
    const int shift = ((lead + skip) & 1) * 16;
#pragma unroll 2
    for (int w = lane; w < words; w += 32) {
      const u32 a = from[2 * w], b = from[2 * w + 1], c = from[2 * w + 2];
      put<true>(Unit<T, 8>{make_uint2(__funnelshift_r(a, b, shift), __funnelshift_r(b, c, shift))}, to + skip + 4 * w, scale, inverse);
    }
    const int i = lane < 4 ? lane : skip + 4 * words + lane - 4;
    if (lane < 4 ? i < skip : lane < 8 && i < row_len) put<false>(Unit<T, 2>{((const unsigned short*)held)[lead + i]}, to + i, scale, inverse);
    __syncwarp();
  }
}

}  // namespace gsb

using namespace gsb;

extern "C" int gsb_quantize_rows(gsb_ctx* ctx, void* stream_, const void* x, int dtype, int64_t num_rows, int64_t row_len, int64_t x_stride,
                                 int8_t* out_values, int64_t values_stride, float* out_scales) {
  GSB_ENTER(ctx);
  const int size = value_bytes(dtype);
  GSB_REQUIRE(num_rows >= 0 && num_rows < ((int64_t)1 << 31) && row_len >= 1 && row_len <= GSB_MAX_ROW_LEN && x_stride >= 0 &&
                  values_stride >= row_len && size != 0,
              GSB_ERR_INVALID_ARGUMENT);
  if (num_rows == 0) return GSB_OK;
  GSB_REQUIRE(x && out_values && out_scales && aligned_to(size, (const char*)x) && aligned_to(4, out_scales), GSB_ERR_INVALID_ARGUMENT);
  cudaStream_t stream = (cudaStream_t)stream_;
  const int unit = unit_bytes(row_len * size, (u64)(uintptr_t)x | (u64)(x_stride * size));
  ScopedKernelTimer timer(ctx, KID_QUANTIZE, stream);
  with_unit(dtype, unit, [&](auto value, auto bytes) {
    typedef decltype(value) T;
    constexpr int B = decltype(bytes)::value;
    constexpr int N = B / (int)sizeof(T);
    constexpr bool can = N == 2 || N == 4 || N == 8;
    const bool packed = can && aligned_to(N, out_values) && values_stride % N == 0;
    const i64 units = row_len * size / B, stride = x_stride * size / B;
    if (units <= 32 * kShortSteps) {  // 459 844 rows of 100 bf16 53 us, a warp a row 112; 500 000 of 64 floats 27 and 139
      int lanes = 1;
      while (lanes * kShortSteps < units) lanes *= 2;
      launch_behind(stream, packed ? k_quantize_short<T, B, can> : k_quantize_short<T, B, false>, grid_for(num_rows, kQuantThreads / lanes * kShortRows),
                    kQuantThreads, (const Unit<T, B>*)x, stride, (int)units, lanes, (u32)num_rows, out_values, values_stride, out_scales);
    } else if (B < 16 && sizeof(T) == 2 && (row_len + 7) / 8 + 1 <= kShiftedRoom) {
      const int room = (int)(row_len + 7) / 8 + 1;
      if constexpr (sizeof(T) == 2)
        launch_behind_with(stream, (size_t)room * 16 * (kQuantThreads / 32), k_quantize_shifted<T>, grid_for(num_rows, kQuantThreads / 32), kQuantThreads,
                           (const T*)x, x_stride, (int)row_len, (u32)num_rows, out_values, values_stride, out_scales, room);
    } else {
      auto* const kernel = units <= 128 ? (packed ? k_quantize_rows<T, B, can, 4> : k_quantize_rows<T, B, false, 4>)
                                        : (packed ? k_quantize_rows<T, B, can, 8> : k_quantize_rows<T, B, false, 8>);
      launch_behind(stream, kernel, grid_for(num_rows, kQuantThreads / 32), kQuantThreads,
                    (const Unit<T, B>*)x, stride, (int)units, (u32)num_rows, out_values, values_stride, out_scales);
    }
  });
  GSB_LAUNCH_OK();
  return GSB_OK;
}
