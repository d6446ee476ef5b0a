// Rows in 8 bits with a scale each: scale[r] = max |x[r, :]| / 127, values[r, :] = x[r, :] / scale[r], rounded to the nearest whole
// number, ties to even.  Divisions are those of IEEE float, so the same rows give the same values wherever that is done.  A row of
// zeros has the scale 0; one that holds an infinity or NaN has a NaN for its scale, and zeros for its values.
#include "launch.cuh"
#include "row_values.cuh"

namespace gsb {

constexpr int kQuantThreads = 256;

__device__ __forceinline__ int quantized(float v, float scale) {
  if (!(scale > 0.f)) return 0;
  return min(127, max(-127, __float2int_rn(__fdiv_rn(v, scale))));
}

// A warp takes a row.
template <class T, int BYTES>
__global__ void __launch_bounds__(kQuantThreads) k_quantize_rows(const Unit<T, BYTES>* __restrict__ x, i64 x_stride, int units, u32 num_rows,
                                                                 int8_t* __restrict__ values, i64 values_stride, float* __restrict__ scales) {
  constexpr int N = Unit<T, BYTES>::N;
  await_previous();
  const int lane = threadIdx.x & 31;
  for (u32 r = (blockIdx.x * kQuantThreads + threadIdx.x) / 32; r < num_rows; r += gridDim.x * (kQuantThreads / 32)) {
    const Unit<T, BYTES>* row = x + (i64)r * x_stride;
    float top = 0.f;
    bool odd = false;
    for (int j = lane; j < units; j += 32) {
      float f[N];
      load_unit(row + j).get(f);
#pragma unroll
      for (int q = 0; q < N; ++q) {
        top = fmaxf(top, fabsf(f[q]));
        odd |= !(fabsf(f[q]) <= 3.402823466e38f);
      }
    }
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    odd = __any_sync(0xffffffffu, odd);
    const float scale = odd ? __int_as_float(0x7fffffff) : __fdiv_rn(top, 127.f);
    if (lane == 0) scales[r] = scale;
    for (int j = lane; j < units; j += 32) {
      float f[N];
      load_unit(row + j).get(f);
      int8_t* to = values + (i64)r * values_stride + (i64)j * N;
#pragma unroll
      for (int q = 0; q < N; ++q) to[q] = (int8_t)quantized(f[q], scale);
    }
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
    const int grid = (int)min((i64)kNumSMs * 8, (i64)grid_for(num_rows, kQuantThreads / 32));
    launch_behind(stream, k_quantize_rows<T, B>, grid, kQuantThreads, (const Unit<T, B>*)x, x_stride * size / B, (int)(row_len * size / B), (u32)num_rows,
                  out_values, values_stride, out_scales);
  });
  GSB_LAUNCH_OK();
  return GSB_OK;
}
