// Host helpers for TMA tensor maps (driver entry point fetched through the runtime, no -lcuda needed).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <torch/extension.h>
#include <c10/cuda/CUDAException.h>

#include <string>

namespace br {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn tma_encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    cudaDriverEntryPointQueryResult q;
    void* ptr = nullptr;
    C10_CUDA_CHECK(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q));
    TORCH_CHECK(q == cudaDriverEntryPointSuccess && ptr, "cuTensorMapEncodeTiled unavailable");
    fn = reinterpret_cast<EncodeTiledFn>(ptr);
  }
  return fn;
}

// 3-D map over storage [dim2][dim1][dim0] (dim0 contiguous) with strides in elements; 128-byte swizzle.
inline CUtensorMap tma_map_3d(CUtensorMapDataType dtype, int elem_bytes, const void* base, int64_t d0, int64_t d1,
                              int64_t d2, int64_t s1, int64_t s2, int box0, int box1,
                              CUtensorMapSwizzle swz = CU_TENSOR_MAP_SWIZZLE_128B) {
  CUtensorMap m;
  if (d2 == 1 || s2 == 0) s2 = s1 * d1;
  cuuint64_t dims[3] = {(cuuint64_t)d0, (cuuint64_t)d1, (cuuint64_t)d2};
  cuuint64_t strides[2] = {(cuuint64_t)(s1 * elem_bytes), (cuuint64_t)(s2 * elem_bytes)};
  cuuint32_t box[3] = {(cuuint32_t)box0, (cuuint32_t)box1, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  TORCH_CHECK(reinterpret_cast<uintptr_t>(base) % 16 == 0, "TMA base must be 16-byte aligned");
  TORCH_CHECK((s1 * elem_bytes) % 16 == 0 && (s2 * elem_bytes) % 16 == 0, "TMA strides must be multiples of 16 bytes");
  CUresult r = tma_encode_fn()(&m, dtype, 3, const_cast<void*>(base), dims, strides, box, estr,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, swz, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed: ", (int)r);
  return m;
}

// Tiles of rows x box_cols elements (64: 128-byte swizzle, 32: 64-byte) of one head of a [rows, heads, D] tensor of 16-bit values (strides in elements,
// multiples of 8): a 3-D map whose dimensions stand in the order of their strides. `swapped`: the coordinates are
// (d, row, head) instead of (d, head, row).
inline CUtensorMap tma_map_head_rows(CUtensorMapDataType dtype, const void* base, int64_t D, int64_t heads, int64_t rows,
                                     int64_t head_stride, int64_t row_stride, int box_rows, bool* swapped, int box_cols = 64) {
  *swapped = head_stride > row_stride;
  CUtensorMap m;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)(*swapped ? rows : heads), (cuuint64_t)(*swapped ? heads : rows)};
  cuuint64_t strides[2] = {(cuuint64_t)(2 * (*swapped ? row_stride : head_stride)),
                           (cuuint64_t)(2 * (*swapped ? head_stride : row_stride))};
  cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)(*swapped ? box_rows : 1), (cuuint32_t)(*swapped ? 1 : box_rows)};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = tma_encode_fn()(&m, dtype, 3, const_cast<void*>(base), dims, strides, box, estr,
                               CU_TENSOR_MAP_INTERLEAVE_NONE,
                               box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed: ", std::to_string((int)r));
  return m;
}

}  // namespace br
