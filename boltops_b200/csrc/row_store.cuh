// 32 consecutive fp32 results of a row on their way to memory (GEMM epilogues).
#pragma once

#include "common.cuh"

namespace bolt {
namespace tc {

// Store 32 consecutive fp32 values as c_dtype starting at column col0 (masked to ncols).
__device__ __forceinline__ void store_row32(void* c, int dt, int64_t row_off, int col0, int ncols,
                                            const float (&v)[32]) {
  if (col0 >= ncols) return;
  const bool full = col0 + 32 <= ncols;
  if (dt == BOLT_F32) {
    float* dst = static_cast<float*>(c) + row_off + col0;
    if (full && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
#pragma unroll
      for (int j = 0; j < 32; j += 4)
        *reinterpret_cast<float4*>(dst + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (col0 + j < ncols) dst[j] = v[j];
    }
    return;
  }
  uint32_t packed[16];
  if (dt == BOLT_BF16) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      packed[j] = *reinterpret_cast<uint32_t*>(&h);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
      packed[j] = *reinterpret_cast<uint32_t*>(&h);
    }
  }
  uint16_t* dst = static_cast<uint16_t*>(c) + row_off + col0;
  if (full && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
#pragma unroll
    for (int j = 0; j < 16; j += 4)
      *reinterpret_cast<uint4*>(dst + 2 * j) =
          make_uint4(packed[j], packed[j + 1], packed[j + 2], packed[j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (col0 + j < ncols) dst[j] = (uint16_t)(packed[j >> 1] >> ((j & 1) * 16));
  }
}

// Pack 32 fp32 values into 64 bytes of bf16 / f16.
__device__ __forceinline__ void pack32_16bit(const float (&v)[32], int dt, uint4 (&w)[4]) {
  uint32_t pk[16];
  if (dt == BOLT_BF16) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      pk[j] = *reinterpret_cast<uint32_t*>(&h);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
      pk[j] = *reinterpret_cast<uint32_t*>(&h);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = make_uint4(pk[4 * j], pk[4 * j + 1], pk[4 * j + 2], pk[4 * j + 3]);
}

}  // namespace tc
}  // namespace bolt
