// Host side of tiled TMA copies: the encoder's entry point and 2-D maps of rows in boxes of 128 bytes with the 128-byte swizzle.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>

#include "jib_kernels.h"

namespace jib {

typedef CUresult (*TmaEncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline TmaEncodeFn tma_encode_fn() {
    static TmaEncodeFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void * p = nullptr;
        cudaDriverEntryPointQueryResult res;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &res) == cudaSuccess && res == cudaDriverEntryPointSuccess)
            fn = (TmaEncodeFn) p;
    });
    return fn;
}

// rows x cols of 1-byte (type UINT8) or 2-byte (BFLOAT16) elements, rows row_bytes apart; a box is 128 bytes wide and box_rows high, zeros outside.
inline int tma_rows_map(CUtensorMap * out, CUtensorMapDataType type, const void * ptr, long long rows, long long cols, long long row_bytes, int box_rows) {
    TmaEncodeFn fn = tma_encode_fn();
    if (!fn) return JIB_E_DRIVER;
    if (((uintptr_t) ptr & 15) || row_bytes % 16) return JIB_E_ALIGN;
    const int el = type == CU_TENSOR_MAP_DATA_TYPE_UINT8 ? 1 : 2;
    const cuuint64_t dims[2] = {(cuuint64_t) cols, (cuuint64_t) rows}, strides[1] = {(cuuint64_t) row_bytes};
    const cuuint32_t box[2] = {(cuuint32_t) (128 / el), (cuuint32_t) box_rows}, step[2] = {1, 1};
    return fn(out, type, 2, const_cast<void *>(ptr), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? 0
               : JIB_E_TENSORMAP;
}

// rows of row_bytes bytes as they are, in boxes box_bytes wide and box_rows high, not swizzled, zeros outside.
inline int tma_bytes_map(CUtensorMap * out, const void * ptr, long long rows, long long row_bytes, int box_bytes, int box_rows) {
    TmaEncodeFn fn = tma_encode_fn();
    if (!fn) return JIB_E_DRIVER;
    if (((uintptr_t) ptr & 15) || row_bytes % 16) return JIB_E_ALIGN;
    const cuuint64_t dims[2] = {(cuuint64_t) row_bytes, (cuuint64_t) rows}, strides[1] = {(cuuint64_t) row_bytes};
    const cuuint32_t box[2] = {(cuuint32_t) box_bytes, (cuuint32_t) box_rows}, step[2] = {1, 1};
    return fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(ptr), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
              CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? 0
               : JIB_E_TENSORMAP;
}

}  // namespace jib
