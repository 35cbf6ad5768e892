// Tensor maps of plain matrices, encoded anew for every call that uses them (a microsecond; nothing is remembered by an address).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ogb {

// [rows, cols] elements of `type`, rows `row_bytes` apart, in boxes of box_rows x box_cols; elements outside read as zero.
inline bool encode_map_2d(CUtensorMap* out, CUtensorMapDataType type, const void* ptr, uint64_t rows, uint64_t cols, uint64_t row_bytes, uint32_t box_rows, uint32_t box_cols,
                          CUtensorMapSwizzle swizzle) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                              CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess ? reinterpret_cast<Encode>(p) : Encode(nullptr);
  }();
  if (!encode) return false;
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {row_bytes};
  const cuuint32_t box[2] = {box_cols, box_rows}, step[2] = {1, 1};
  return encode(out, type, 2, const_cast<void*>(ptr), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace ogb
