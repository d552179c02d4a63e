// Rows of fp32 in shared memory as the exact kernels on CUDA cores hold and multiply them.
#pragma once

#include <cuda_runtime.h>

namespace pjx {

// Elements between two rows of `d` elements: whole 16 bytes, and one more, so that rows start in different banks.
__host__ __device__ inline int pitch4(int d) { return (d + 3) / 4 * 4 + 4; }
__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float dot4(float4 a, float4 b, float s) {
  return fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, fmaf(a.x, b.x, s))));
}

}  // namespace pjx
