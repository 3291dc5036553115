// Operands in fp32, bf16 or fp16: the kernels that take all three read them into fp32 registers, compute there, and round
// once where they store.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace nb200 {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// N neighbouring values as they lie in memory (16-byte accesses where N values are 16 bytes or a multiple of it)
template <typename T, int N> struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack {
  T v[N];
  // Value i in fp32. Of 16-bit pairs by words: taken one by one they cost an instruction more each to pick them out.
  __device__ __forceinline__ float f(int i) const {
    if constexpr (N % 2 == 0 && std::is_same<T, __nv_bfloat16>::value) {
      const uint32_t w = reinterpret_cast<const uint32_t *>(v)[i / 2];
      return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    } else if constexpr (N % 2 == 0 && std::is_same<T, __half>::value) {
      const __half2 h = reinterpret_cast<const __half2 *>(v)[i / 2];
      return i & 1 ? __high2float(h) : __low2float(h);
    } else {
      return to_f32(v[i]);
    }
  }
  __device__ __forceinline__ void fill(float f) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = from_f32<T>(f);
  }
  __device__ __forceinline__ void clear() {
    if constexpr (N * sizeof(T) % 4 == 0) {
#pragma unroll
      for (int i = 0; i < (int)(N * sizeof(T) / 4); ++i)
        reinterpret_cast<uint32_t *>(v)[i] = 0u;
    } else {
      fill(0.0f);
    }
  }
};
template <typename T, int N> __device__ __forceinline__ Pack<T, N> load_pack(const T *p) {
  return *reinterpret_cast<const Pack<T, N> *>(p);
}
// The same for data that this pass reads once. In program order (volatile): a run of them is in flight together, where the
// compiler would otherwise put each next to its use to save registers.
template <typename T, int N> __device__ __forceinline__ Pack<T, N> load_pack_stream(const T *p) {
  if constexpr (N * sizeof(T) == 16) {
    uint4 u;
    asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
    return *reinterpret_cast<const Pack<T, N> *>(&u);
  } else {
    return load_pack<T, N>(p);
  }
}
// Rounding of neighbouring values, two at a time where the type has it.
template <typename T, int N> __device__ __forceinline__ Pack<T, N> round_pack(const float (&v)[N]) {
  Pack<T, N> o;
  if constexpr (N % 2 == 0 && std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
    for (int i = 0; i < N; i += 2)
      *reinterpret_cast<__nv_bfloat162 *>(&o.v[i]) = __floats2bfloat162_rn(v[i], v[i + 1]);
  } else if constexpr (N % 2 == 0 && std::is_same<T, __half>::value) {
#pragma unroll
    for (int i = 0; i < N; i += 2)
      *reinterpret_cast<__half2 *>(&o.v[i]) = __floats2half2_rn(v[i], v[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      o.v[i] = from_f32<T>(v[i]);
  }
  return o;
}
template <typename T, int N> __device__ __forceinline__ void store_pack(T *p, const float (&v)[N], bool keep = true) {
  const Pack<T, N> o = round_pack<T, N>(v);
  if constexpr (N * sizeof(T) == 16)
    st_result(reinterpret_cast<uint4 *>(p), *reinterpret_cast<const uint4 *>(&o), keep);
  else
    *reinterpret_cast<Pack<T, N> *>(p) = o;
}

template <typename T> constexpr int kPackOf = (int)(16 / sizeof(T)); // values in 16 bytes

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1)
    v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1)
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

// Calls f(T{}) with the C++ type of an NB200_F32 / _BF16 / _F16 code.
template <typename F> int with_type(int code, F f) {
  switch (code) {
  case NB200_F32: return f(float{});
  case NB200_BF16: return f(__nv_bfloat16{});
  case NB200_F16: return f(__half{});
  }
  return fail(NB200_EVALUE, "unknown type code %d", code);
}
inline size_t type_bytes(int code) { return code == NB200_F32 ? 4 : 2; }
inline bool aligned8(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 7) == 0; }
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

} // namespace nb200
