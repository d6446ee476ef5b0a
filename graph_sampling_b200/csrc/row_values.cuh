// Rows of float, half or bfloat16 values read and written in units of 16, 8, 4 or 2 bytes, with the arithmetic in float.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace gsb {

template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <int BYTES>
struct WordOf;
template <>
struct WordOf<16> { typedef uint4 type; };
template <>
struct WordOf<8> { typedef uint2 type; };
template <>
struct WordOf<4> { typedef u32 type; };
template <>
struct WordOf<2> { typedef unsigned short type; };

// BYTES of a row: one access each way.  Held as the words they are; the N values exist only where they are worked with (an
// array of 16-bit values does not stay in registers).
template <class T, int BYTES>
struct Unit {
  typedef typename WordOf<BYTES>::type Word;
  static constexpr int N = BYTES / (int)sizeof(T);
  Word w;

  __device__ __forceinline__ void get(float (&f)[N]) const {
    if constexpr (BYTES == 2) {
      f[0] = std::is_same<T, __half>::value ? __half2float(__ushort_as_half(w)) : __uint_as_float((u32)w << 16);
    } else {
      u32 q[BYTES / 4];
      words(q);
#pragma unroll
      for (int i = 0; i < BYTES / 4; ++i) {
        if constexpr (sizeof(T) == 4) {
          f[i] = __uint_as_float(q[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
          f[2 * i] = __half2float(__ushort_as_half((unsigned short)q[i]));
          f[2 * i + 1] = __half2float(__ushort_as_half((unsigned short)(q[i] >> 16)));
        } else {
          f[2 * i] = __uint_as_float(q[i] << 16);
          f[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
        }
      }
    }
  }
  // Rounds to nearest even.
  __device__ __forceinline__ void set(const float (&f)[N]) {
    if constexpr (BYTES == 2) {
      w = bits(f[0]);
    } else {
      u32 q[BYTES / 4];
#pragma unroll
      for (int i = 0; i < BYTES / 4; ++i) {
        if constexpr (sizeof(T) == 4) q[i] = __float_as_uint(f[i]);
        else q[i] = (u32)bits(f[2 * i]) | (u32)bits(f[2 * i + 1]) << 16;
      }
      if constexpr (BYTES == 4) w = q[0];
      else if constexpr (BYTES == 8) w = make_uint2(q[0], q[1]);
      else w = make_uint4(q[0], q[1], q[2], q[3]);
    }
  }
  __device__ __forceinline__ void clear() {
    if constexpr (BYTES <= 4) w = 0;
    else if constexpr (BYTES == 8) w = make_uint2(0, 0);
    else w = make_uint4(0, 0, 0, 0);
  }

 private:
  __device__ __forceinline__ void words(u32 (&q)[BYTES / 4 > 0 ? BYTES / 4 : 1]) const {
    if constexpr (BYTES == 4) q[0] = w;
    else if constexpr (BYTES == 8) q[0] = w.x, q[1] = w.y;
    else q[0] = w.x, q[1] = w.y, q[2] = w.z, q[3] = w.w;
  }
  static __device__ __forceinline__ unsigned short bits(float f) {
    if constexpr (std::is_same<T, __half>::value) return __half_as_ushort(__float2half_rn(f));
    else return __bfloat16_as_ushort(__float2bfloat16_rn(f));
  }
};

template <class T, int BYTES>
__device__ __forceinline__ Unit<T, BYTES> load_unit(const Unit<T, BYTES>* p) {
  return Unit<T, BYTES>{__ldg((const typename WordOf<BYTES>::type*)p)};
}
// What is read once and not again soon.
template <class T, int BYTES>
__device__ __forceinline__ Unit<T, BYTES> load_unit_once(const Unit<T, BYTES>* p) {
  return Unit<T, BYTES>{__ldcs((const typename WordOf<BYTES>::type*)p)};
}
template <class T, int BYTES>
__device__ __forceinline__ void store_unit(Unit<T, BYTES>* p, const Unit<T, BYTES>& u) {
  *(typename WordOf<BYTES>::type*)p = u.w;
}

// What is written and not read soon.
template <class T, int BYTES>
__device__ __forceinline__ void store_unit_once(Unit<T, BYTES>* p, const Unit<T, BYTES>& u) {
  __stcs((typename WordOf<BYTES>::type*)p, u.w);
}

inline int value_bytes(int dtype) { return dtype == GSB_F32 ? 4 : dtype == GSB_F16 || dtype == GSB_BF16 ? 2 : 0; }

// The largest unit that divides a row and every address a row can start at: `addresses` is the bitwise or of base pointers
// and row strides in bytes.
inline int unit_bytes(int64_t row_bytes, uint64_t addresses) {
  const uint64_t all = (uint64_t)row_bytes | addresses;
  return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
}

// Every address is a multiple of `bytes` (null is).
template <class... P>
bool aligned_to(int bytes, const P*... p) {
  return (((uint64_t)(uintptr_t)p | ...) & (uint64_t)(bytes - 1)) == 0;
}

// How a row is taken: by `lanes` neighbouring lanes (a power of two up to 32), `steps` units (1 .. 4) of each at a time.  Of the shapes
// that take the row at once the one that leaves the fewest lanes idle; among equals the one whose steps are nearest to
// `wanted`.  Rows of more than 96 units go in tiles of 32 lanes with `wide` units each.
struct RowShape {
  int lanes, steps;
};
inline RowShape row_shape(int64_t units, int wanted, int wide) {
  RowShape best{32, wide};
  if (units > 96) return best;
  int idle = 1 << 20, away = 0;
  for (int lanes = 32; lanes >= 1; lanes /= 2) {
    const int steps = (int)((units + lanes - 1) / lanes), rest = lanes * steps - (int)units;
    const int off = steps > wanted ? steps - wanted : wanted - steps;
    if (steps <= 4 && (rest < idle || (rest == idle && off < away))) {
      idle = rest;
      away = off;
      best = RowShape{lanes, steps};
    }
  }
  return best;
}
// What copies and combines rows does well with two units of 16 bytes a lane, or four smaller ones (65 528 rows of 2 KB combined in 28
// us, with one unit a lane in 34; 314 602 rows of 200 bytes in 26, with two units of 8 bytes in 30); what sums them, which has
// more to do per row and lane, with one of 16 bytes or four of 4 (1 000 003 rows of 256 bytes 81 us, with two units 96; 1.3 M
// rows of 100 bytes 51, with one unit 83).
inline int copy_steps(int unit) { return unit == 16 ? 2 : 4; }
inline int sum_steps(int unit) { return unit >= 16 ? 1 : unit == 8 ? 2 : 4; }
// Of long rows: four narrow units, though the last tile leaves more lanes idle (50 000 tokens to 200 000 rows of 1 434 bf16: spread 209
// us for 258, combined 207 for 252; 200 000 rows of 602 looked up 86 for 92, summed 150 for 168), but two of 16 bytes (200 000 rows
// of 2 KB combined 89 us, with four 95), and of 8 where they are summed (few rows of 602 floats 131 us, with four 140).
inline int copy_wide(int unit) { return unit == 16 ? 2 : 4; }
inline int sum_wide(int unit) { return unit >= 8 ? 2 : 4; }
// Rows that a group of lanes has on their way at once.  More of them cost warps: with twice as many 65 528 rows of 2 KB were spread
// in 29 us for 25, 314 602 of 200 bytes in 33 for 26.
constexpr int rows_ahead(int steps) { return steps == 1 ? 4 : 2; }

template <class F>
void with_steps(int steps, F f) {
  using std::integral_constant;
  if (steps == 1) f(integral_constant<int, 1>{});
  else if (steps == 2) f(integral_constant<int, 2>{});
  else if (steps == 3) f(integral_constant<int, 3>{});
  else f(integral_constant<int, 4>{});
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
