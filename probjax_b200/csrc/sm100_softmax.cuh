// The softmax of a row of scores that lies in tensor memory, as the tcgen05 attention kernels take it: one thread per row.
#pragma once

#include "pjx_common.cuh"
#include "sm100_ptx.cuh"

namespace pjx {
namespace sm100 {

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (BF16) {
    __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&t);
  } else {
    __half2 t = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&t);
  }
}

// p = exp2(x * cs - m) for one row of BN scores, running sums, pack to 16 bits and
// store over the scores in tensor memory. All exponentials of the row form one
// straight-line block (the stores come last) so that the scheduler can overlap the
// latencies of independent elements.
template <int BN, bool BF16>
__device__ __forceinline__ void exp_pack_store(const float (&s)[BN], float2 cs2, float2 nm2, float2& sum0,
                                               float2& sum1, uint32_t s_addr) {
  uint32_t pk[BN / 2];
#pragma unroll
  for (int i = 0; i < BN / 2; i += 2) {
    const float2 x0 = __ffma2_rn(make_float2(s[2 * i], s[2 * i + 1]), cs2, nm2);
    const float2 x1 = __ffma2_rn(make_float2(s[2 * i + 2], s[2 * i + 3]), cs2, nm2);
    const float2 p0 = make_float2(ex2_approx(x0.x), ex2_approx(x0.y));
    const float2 p1 = make_float2(ex2_approx(x1.x), ex2_approx(x1.y));
    sum0 = __fadd2_rn(sum0, p0);
    sum1 = __fadd2_rn(sum1, p1);
    pk[i] = pack16<BF16>(p0.x, p0.y);
    pk[i + 1] = pack16<BF16>(p1.x, p1.y);
  }
#pragma unroll
  for (int c = 0; c < BN / 64; ++c) tmem_st32(s_addr + c * 32, *reinterpret_cast<const uint32_t(*)[32]>(&pk[c * 32]));
}

}  // namespace sm100
}  // namespace pjx
