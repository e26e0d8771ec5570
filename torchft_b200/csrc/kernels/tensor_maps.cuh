// Tensor maps of bf16 matrices for TMA copies in boxes with a 128- or 64-byte swizzle.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "ftb200_common.cuh"

namespace ftb200 {

// The driver's entry, looked for once; of several first calls at once all wait for the answer.
inline PFN_cuTensorMapEncodeTiled_v12000 encode_tiled() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult qres;
    const bool found = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qres) == cudaSuccess &&
                       qres == cudaDriverEntryPointSuccess;
    return found ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(sym) : nullptr;
  }();
  return fn;
}

template <int N>
int encode_bf16(CUtensorMap* map, const void* base, const cuuint64_t (&gdim)[N], const cuuint64_t (&gstride)[N - 1], const cuuint32_t (&box)[N],
                CUtensorMapSwizzle swizzle) {
  const auto fn = encode_tiled();
  if (fn == nullptr) return FTB200_E_DRIVER;
  cuuint32_t estr[N];
  for (int i = 0; i < N; ++i) estr[i] = 1;
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, N, const_cast<void*>(base), gdim, gstride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : FTB200_E_DRIVER;
}

// [rows, cols] view with row stride ld (elements)
inline int encode_2d(CUtensorMap* map, const void* base, long long rows, long long cols, long long ld, int box_cols, int box_rows) {
  const cuuint64_t gdim[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t gstride[1] = {static_cast<cuuint64_t>(ld) * 2};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
  return encode_bf16(map, base, gdim, gstride, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// [batch, seq, cols] view with row stride ld (elements), the sequence as a dimension of its own; boxes of 32 columns have a swizzle as wide as they are
inline int encode_rows(CUtensorMap* map, const void* base, long long batch, long long seq, long long cols, long long ld, unsigned box_cols = 64,
                       unsigned box_rows = 128) {
  const cuuint64_t gdim[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(seq), static_cast<cuuint64_t>(batch)};
  const cuuint64_t gstride[2] = {static_cast<cuuint64_t>(ld) * 2, static_cast<cuuint64_t>(seq) * ld * 2};
  const cuuint32_t box[3] = {box_cols, box_rows, 1u};
  return encode_bf16(map, base, gdim, gstride, box, box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

}  // namespace ftb200
