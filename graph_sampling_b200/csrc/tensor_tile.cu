// Descriptions of arrays for TMA loads, made on the host.  The driver's function is asked for through the runtime: the library is not
// linked with the driver's.
#include "tensor_tile.cuh"

namespace gsb {

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
  static const EncodeTiled found = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult status;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &status) != cudaSuccess ||
        status != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return (EncodeTiled)fn;
  }();
  return found;
}

// The driver's call wants the device's context to be current on this thread, which only calls of the runtime make it: a thread of autograd's that
// comes here first has none yet.
template <class F>
static bool encoded(F encode) {
  if (encode() == CUDA_SUCCESS) return true;
  int device;
  return cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess && encode() == CUDA_SUCCESS;
}

bool describe_array(CUtensorMap* map, const void* base, int value_bytes, int rank, const u64* dims, const u64* strides, const u32* box,
                    bool swizzled) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return false;
  cuuint64_t extents[5], distances[4];
  cuuint32_t boxes[5], ones[5] = {1, 1, 1, 1, 1};
  for (int d = 0; d < rank; ++d) {
    extents[d] = dims[d];
    boxes[d] = box[d];
    if (d > 0) distances[d - 1] = strides[d - 1];
  }
  return encoded([&] {
    return encode(map, value_bytes == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(base), extents,
                  distances, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
}

bool describe_rows(CUtensorMap* map, void* base, int value_bytes, u64 width, u64 rows) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return false;
  const cuuint64_t extents[2] = {width, rows}, distance[1] = {width * (u64)value_bytes};
  const cuuint32_t box[2] = {64u / (u32)value_bytes, 32}, ones[2] = {1, 1};
  return encoded([&] {
    return encode(map, value_bytes == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, extents, distance, box, ones,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
}

}  // namespace gsb
