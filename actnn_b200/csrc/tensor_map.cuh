// Tensor maps of matrices, made on the host for one call.
#pragma once

#include <atomic>

#include <cuda.h>

#include "common.cuh"

namespace actnn {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiled encode_tiled() {
  static std::atomic<EncodeTiled> fn{nullptr};
  EncodeTiled f = fn.load(std::memory_order_acquire);
  if (!f) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    f = (EncodeTiled)p;
    fn.store(f, std::memory_order_release);
  }
  return f;
}
// Rows of `cols` bytes, `ld` bytes apart, in boxes of `wide` bytes by `high` rows, zeros where a box reaches past the matrix; swizzled in
// lines of 128 bytes, or as they are.
inline bool map_bytes(CUtensorMap* m, const void* p, int64_t cols, int64_t rows, int64_t ld, int wide, int high, bool swizzled) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
  const cuuint32_t boxes[2] = {(cuuint32_t)wide, (cuuint32_t)high}, ones[2] = {1, 1};
  const EncodeTiled f = encode_tiled();
  return f && f(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Values [rows, cols] of a type, contiguous, in boxes.
inline bool map_values(CUtensorMap* m, void* p, int64_t cols, int64_t rows, int dtype, int wide, int high) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(cols * dtype_size(dtype))};
  const cuuint32_t boxes[2] = {(cuuint32_t)wide, (cuuint32_t)high}, ones[2] = {1, 1};
  const CUtensorMapDataType type = dtype == ACTNN_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dtype == ACTNN_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const EncodeTiled f = encode_tiled();
  return f && f(m, type, 2, p, dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace actnn
