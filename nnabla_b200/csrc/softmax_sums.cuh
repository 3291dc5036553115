// The running maximum and sum of a softmax.
#pragma once
#include "typed.cuh"

namespace nb200 {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float v) { // 2^v; results below 2^-126 are zero
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Maximum and sum of 2^((v - maximum) * scale). A maximum of -infinity has the sum 0.
struct MaxSum {
  float m, s;
};
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float scale) {
  const float m = fmaxf(a.m, b.m), base = m == -INFINITY ? 0.0f : m;
  return {m, a.s * ex2((a.m - base) * scale) + b.s * ex2((b.m - base) * scale)};
}
__device__ __forceinline__ MaxSum warp_join(MaxSum v, float scale) {
#pragma unroll
  for (int d = 16; d; d >>= 1)
    v = join(v, MaxSum{__shfl_xor_sync(0xffffffffu, v.m, d), __shfl_xor_sync(0xffffffffu, v.s, d)}, scale);
  return v;
}

} // namespace nb200
