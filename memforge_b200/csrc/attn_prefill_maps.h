// Tensor maps of the tcgen05 chunk kernel.
#pragma once

#include "mf_internal.h"

namespace mf {

typedef CUresult (*EncodeTiledFn2)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn2 encode_fn() {
  static EncodeTiledFn2 fn = []() -> EncodeTiledFn2 {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<EncodeTiledFn2>(ptr);
  }();
  return fn;
}

// 4-D view (64 elements, dim1, 2 halves of 64, dim3) with byte strides
// (s1, 128, s3) and box (64, b1, 1, b3), 128-byte swizzle.
static CUresult encode_pf(CUtensorMap* m, const void* base, uint64_t n1, uint64_t s1,
                          uint64_t n3, uint64_t s3, uint32_t b1, uint32_t b3,
                          CUtensorMapDataType dt) {
  EncodeTiledFn2 fn = encode_fn();
  if (!fn) return CUDA_ERROR_NOT_SUPPORTED;
  cuuint64_t dims[4] = {64, n1, 2, n3};
  cuuint64_t strides[3] = {s1, 128, s3};
  cuuint32_t box[4] = {64, b1, 1, b3};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(m, dt, 4, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

}  // namespace mf
