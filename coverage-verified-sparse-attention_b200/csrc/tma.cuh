// Tensor copies (TMA): the map of a [tokens, heads, D] array of 16-bit elements, and the
// copy of one of its tiles into this CTA's shared memory, 128-byte swizzle.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cvsa_common.cuh"

namespace cvsa {

// Tiles of `tokens` tokens of `heads` heads of 64 elements. False where the array's strides
// or sizes are none that a map takes.
inline bool token_map(CUtensorMap* map, const void* p, bool bf16, int64_t n_tokens, int64_t n_heads,
                      int d, int64_t token_stride, int64_t head_stride, int tokens, int heads) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                              CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                              CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) !=
            cudaSuccess || found != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return reinterpret_cast<Encode>(fn);
  }();
  if (!encode || token_stride <= 0 || head_stride <= 0) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)n_heads, (cuuint64_t)n_tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)token_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)heads, (cuuint32_t)tokens}, step[3] = {1, 1, 1};
  return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The tile whose first element is (token, head, x), x a multiple of 8; parts of it past
// the array are zeros. One thread; completes on `bar` with the tile's bytes.
__device__ __forceinline__ void token_load(uint32_t dst, const CUtensorMap* map, int x, int head,
                                           int token, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(head), "r"(token), "r"(smem_u32(bar))
      : "memory");
}

}  // namespace cvsa
