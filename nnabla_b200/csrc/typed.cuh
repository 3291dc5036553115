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

// N neighbouring values as they lie in memory (16-byte accesses where N values are 16 bytes or a multiple of it), kept as words
// where they fill some: 16-bit values that are picked out one by one cost an instruction or two more each.
template <typename T, int N> struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack {
  static constexpr bool kWords = N * sizeof(T) % 4 == 0;
  static constexpr int kPer = sizeof(T) == 4 || !kWords ? 1 : 2; // values a word
  std::conditional_t<kWords, uint32_t, uint16_t> w[N / kPer];
  __device__ __forceinline__ float f(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      return kPer == 1 ? __uint_as_float((uint32_t)w[i] << 16)
                       : __uint_as_float(i & 1 ? w[i / kPer] & 0xffff0000u : (uint32_t)w[i / kPer] << 16);
    } else if constexpr (kPer == 1) {
      return __half2float(__ushort_as_half(w[i]));
    } else {
      const __half2 h = *reinterpret_cast<const __half2 *>(&w[i / 2]);
      return i & 1 ? __high2float(h) : __low2float(h);
    }
  }
  __device__ __forceinline__ void set(int i, T v) {
    if constexpr (sizeof(T) == 4) {
      w[i] = *reinterpret_cast<const uint32_t *>(&v);
    } else {
      const uint32_t b = *reinterpret_cast<const uint16_t *>(&v);
      if constexpr (kPer == 1)
        w[i] = (uint16_t)b;
      else
        w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | b << 16 : (w[i / 2] & 0xffff0000u) | b;
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < N / kPer; ++i)
      w[i] = 0;
  }
  __device__ __forceinline__ void fill(float f) {
    clear();
#pragma unroll
    for (int i = 0; i < N; ++i)
      set(i, from_f32<T>(f));
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
  if constexpr (sizeof(T) == 2 && N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[i], v[i + 1]);
        o.w[i / 2] = *reinterpret_cast<const uint32_t *>(&h);
      } else {
        const __half2 h = __floats2half2_rn(v[i], v[i + 1]);
        o.w[i / 2] = *reinterpret_cast<const uint32_t *>(&h);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      o.set(i, from_f32<T>(v[i]));
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

// Asynchronous copies to shared memory, in groups: cp_async_wait<N> waits until at most N of this thread's groups are under way.
__device__ __forceinline__ void cp_async16(void *to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

} // namespace nb200
