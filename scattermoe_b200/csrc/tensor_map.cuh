// Host-side tensor maps for the streaming kernels: 16-bit elements, up to five axes.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace smoe {

typedef CUresult (*TensorMapEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                      const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                      CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder, looked up once (the library does not link against the driver).
inline TensorMapEncodeFn tensor_map_encoder() {
  static TensorMapEncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<TensorMapEncodeFn>(p);
  }();
  return fn;
}

// Axis 0 is contiguous; `stride[i]` of axis i + 1 in bytes (multiples of 16). Elements outside the axes read as zero.
inline bool encode_tensor_map(CUtensorMap* map, bool bf16, const void* base, int rank, const uint64_t* dim, const uint64_t* stride,
                              const uint32_t* box, CUtensorMapSwizzle swizzle,
                              CUtensorMapL2promotion promotion = CU_TENSOR_MAP_L2_PROMOTION_L2_256B) {
  TensorMapEncodeFn fn = tensor_map_encoder();
  if (!fn) return false;
  cuuint64_t dims[5], strides[4];
  cuuint32_t boxes[5], step[5];
  for (int i = 0; i < rank; ++i) {
    dims[i] = dim[i];
    boxes[i] = box[i];
    step[i] = 1;
    if (i + 1 < rank) strides[i] = stride[i];
  }
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, static_cast<cuuint32_t>(rank),
            const_cast<void*>(base), dims, strides, boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
            promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace smoe
