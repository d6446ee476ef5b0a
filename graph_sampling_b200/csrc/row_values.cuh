// Rows of float, half or bfloat16 values read and written in units of 16, 8, 4 or 2 bytes, with the arithmetic in float.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace gsb {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// BYTES of a row as N values: one access each way.
template <class T, int BYTES>
struct alignas(BYTES) Unit {
  static constexpr int N = BYTES / (int)sizeof(T);
  T v[N];
};

template <int BYTES>
struct Word;
template <>
struct Word<16> { typedef uint4 type; };
template <>
struct Word<8> { typedef uint2 type; };
template <>
struct Word<4> { typedef unsigned int type; };
template <>
struct Word<2> { typedef unsigned short type; };

template <class T, int BYTES>
__device__ __forceinline__ Unit<T, BYTES> load_unit(const Unit<T, BYTES>* p) {
  typedef typename Word<BYTES>::type W;
  union {
    W w;
    Unit<T, BYTES> u;
  } x;
  x.w = __ldg((const W*)p);
  return x.u;
}
// What is read once and not again soon, and what is written and not read soon.
template <class T, int BYTES>
__device__ __forceinline__ Unit<T, BYTES> load_unit_once(const Unit<T, BYTES>* p) {
  typedef typename Word<BYTES>::type W;
  union {
    W w;
    Unit<T, BYTES> u;
  } x;
  x.w = __ldcs((const W*)p);
  return x.u;
}
template <class T, int BYTES>
__device__ __forceinline__ void store_unit(Unit<T, BYTES>* p, const Unit<T, BYTES>& u) {
  typedef typename Word<BYTES>::type W;
  union {
    W w;
    Unit<T, BYTES> u;
  } x;
  x.u = u;
  *(W*)p = x.w;
}
template <class T, int BYTES>
__device__ __forceinline__ void store_unit_once(Unit<T, BYTES>* p, const Unit<T, BYTES>& u) {
  typedef typename Word<BYTES>::type W;
  union {
    W w;
    Unit<T, BYTES> u;
  } x;
  x.u = u;
  __stcs((W*)p, x.w);
}

inline int value_bytes(int dtype) { return dtype == GSB_F32 ? 4 : dtype == GSB_F16 || dtype == GSB_BF16 ? 2 : 0; }

// The largest unit that divides a row and every address a row can start at: `addresses` is the bitwise or of base pointers
// and row strides in bytes.
inline int unit_bytes(int64_t row_bytes, uint64_t addresses) {
  const uint64_t all = (uint64_t)row_bytes | addresses;
  return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
}

// Calls f(T, integral_constant<int, BYTES>) for the value type and the unit.
template <class F>
void with_unit(int dtype, int unit, F f) {
  using std::integral_constant;
  auto by_unit = [&](auto value) {
    if (unit == 16) f(value, integral_constant<int, 16>{});
    else if (unit == 8) f(value, integral_constant<int, 8>{});
    else if (unit == 4) f(value, integral_constant<int, 4>{});
    else if constexpr (sizeof(value) == 2) f(value, integral_constant<int, 2>{});
  };
  if (dtype == GSB_F32) by_unit(float{});
  else if (dtype == GSB_F16) by_unit(__half{});
  else by_unit(__nv_bfloat16{});
}

}  // namespace gsb
