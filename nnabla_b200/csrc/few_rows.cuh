// The classifying head for up to eight rows: W decides, 2 or 4 bytes for every two to sixteen operations a row, so that the
// CUDA cores in fp32 keep up with HBM and nothing is laid out first.
#pragma once
#include "loss_gemm.cuh"

namespace nb200 {

constexpr int kFewRows = 8;
constexpr int kFewThreads = 256, kFewValues = 8192; // of x held in shared memory at a time

constexpr int kFewBatch = 4, kFewBatches = 3;                         // packs a group of copies, groups on the way
constexpr int kFewRing = kFewBatch * kFewBatches * kFewThreads * 16; // bytes

template <typename T, int VEC> constexpr int few_lanes() { return VEC * sizeof(T) == 16 ? 4 : 32; }

__device__ __forceinline__ void cp_async16(void *to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ptx::smem_u32(to)), "l"(from) : "memory");
}
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// l = x W + b for a few classes a block: 64 bytes of a row of W, four lanes, eight rows a warp, so that the blocks are many and
// their rounds even (with 128 bytes 500 blocks for 32000 classes, 4 on some SMs and 3 on others: 28 us); 32 lanes of one value
// where rows do not begin at 16-byte boundaries. Of those sums
// kSums leaves the maximum and the sum of the exponentials, kGrad G in fp32.
template <typename T, int R, int VEC, Out kOut>
__global__ void __launch_bounds__(kFewThreads) few_logits_kernel(const T *__restrict__ x, const T *__restrict__ w,
                                                                 const T *__restrict__ bias, LossRows rows, int count,
                                                                 int64_t size, float *__restrict__ g, int64_t ldg) {
  constexpr bool kAsync = VEC * sizeof(T) == 16;
  constexpr int kLanes = few_lanes<T, VEC>(), kCols = kLanes * VEC, kStep = kFewThreads / kLanes; // kStep: rows of W a pass
  constexpr int kFewK = kFewValues / R;
  extern __shared__ __align__(16) uint8_t few_smem[];
  uint4(*ring)[kFewThreads] = reinterpret_cast<uint4(*)[kFewThreads]>(few_smem); // [kFewBatches * kFewBatch]
  float *xs = reinterpret_cast<float *>(few_smem + (kAsync ? kFewRing : 0));
  float(*sums)[R][kCols] = reinterpret_cast<float(*)[R][kCols]>(few_smem); // in the same place, behind the last use of both
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t classes = rows.classes, c0 = (int64_t)blockIdx.x * kCols, c = c0 + (threadIdx.x % kLanes) * VEC;
  const bool here = c < classes; // (VEC divides classes, or is 1)
  float acc[R][VEC];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      acc[r][j] = 0.0f;
  // W by asynchronous copies, each thread for itself: kFewBatches groups of kFewBatch packs on the way, whatever the compiler
  // makes of the registers (with eight ordinary loads a step it kept few in flight: 3.4 TB/s). A thread's rows of W are
  // (threadIdx.x / kLanes) + kStep * i through all pieces of K, kFewK being a multiple of kFewBatch * kStep.
  static_assert(!kAsync || kFewK % (kFewBatch * kStep) == 0, "a piece of K is whole groups");
  int64_t next = threadIdx.x / kLanes;
  int fetched = 0, batch = 0;
  auto fetch = [&]() {
    if constexpr (kAsync) {
      const int at = fetched++ % kFewBatches * kFewBatch;
#pragma unroll
      for (int u = 0; u < kFewBatch; ++u, next += kStep)
        if (here && next < size)
          cp_async16(&ring[at + u][threadIdx.x], w + next * classes + c);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  if constexpr (kAsync)
    for (int i = 0; i < kFewBatches; ++i)
      fetch();
  for (int64_t k0 = 0; k0 < size; k0 += kFewK) {
    const int n = (int)(size - k0 < kFewK ? size - k0 : kFewK);
    if (k0)
      __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll 4
      for (int k = threadIdx.x; k < n; k += kFewThreads)
        xs[k * R + r] = r < count ? to_f32(x[r * size + k0 + k]) : 0.0f;
    __syncthreads();
    if (!here)
      continue;
    auto add = [&](const Pack<T, VEC> &v, int k) {
      float xv[R];
#pragma unroll
      for (int r = 0; r < R; ++r)
        xv[r] = xs[k * R + r];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          acc[r][j] = fmaf(xv[r], v.f(j), acc[r][j]);
    };
    if constexpr (kAsync) {
      for (int k = threadIdx.x / kLanes; k < n; k += kFewBatch * kStep) {
        const int at = batch % kFewBatches * kFewBatch;
        cp_async_wait<kFewBatches - 1>();
#pragma unroll
        for (int u = 0; u < kFewBatch; ++u)
          if (k + u * kStep < n)
            add(*reinterpret_cast<const Pack<T, VEC> *>(&ring[at + u][threadIdx.x]), k + u * kStep);
        fetch();
        ++batch;
      }
    } else {
      for (int k = threadIdx.x / kLanes; k < n; k += kStep)
        add(load_pack<T, VEC>(w + (k0 + k) * classes + c), k);
    }
  }
  if constexpr (kAsync)
    cp_async_wait<0>();
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float s = acc[r][j];
#pragma unroll
      for (int d = 16; d >= kLanes; d >>= 1)
        s += __shfl_xor_sync(0xffffffffu, s, d);
      if (lane < kLanes)
        sums[warp][r][lane * VEC + j] = s;
    }
  __syncthreads();
  for (int r = warp; r < count; r += kFewThreads / 32) { // a warp a row
    const int64_t label = rows.label_of(r);
    MaxSum t{-INFINITY, 0.0f};
    for (int i = lane; i < kCols; i += 32) {
      if (c0 + i >= classes)
        continue;
      float l = 0.0f;
#pragma unroll
      for (int u = 0; u < kFewThreads / 32; ++u)
        l += sums[u][r][i];
      if (bias)
        l += to_f32(bias[c0 + i]);
      if constexpr (kOut == Out::kSums) {
        t = join(t, MaxSum{l, l == -INFINITY ? 0.0f : l != l ? l : 1.0f}, kLog2e);
        if (c0 + i == label)
          rows.target[r] = l;
      } else {
        const float2 st = rows.stat[r];
        const float v = ex2(fmaf(l - st.x, kLog2e, -st.y * kLog2e)) - (c0 + i == label ? 1.0f : 0.0f);
        g[r * ldg + c0 + i] = label < 0 ? 0.0f : label >= classes ? NAN : v * rows.dloss[r];
      }
    }
    if constexpr (kOut == Out::kSums) {
      t = warp_join(t, kLog2e);
      if (lane == 0)
        rows.partial[(int64_t)r * rows.tiles + blockIdx.x] = make_float2(t.m, t.s);
    }
  }
}

// dx = G W^T and dW = x^T G in one pass over W: a block has kFewH rows of W, its threads walk along the classes. A pack of
// G, [R][VEC] in fp32 from L2, serves all of the block's rows.
constexpr int kFewH = 4;
template <typename T, int R, int VEC>
__global__ void __launch_bounds__(kFewThreads) few_grads_kernel(const T *__restrict__ x, const T *__restrict__ w,
                                                                const float *__restrict__ g, int64_t ldg, T *dx, T *dw,
                                                                int count, int64_t size, int64_t classes, bool accum_dx,
                                                                bool accum_dw, bool keep) {
  __shared__ float sums[kFewThreads / 32][kFewH * R];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t h0 = (int64_t)blockIdx.x * kFewH;
  const int hs = (int)(size - h0 < kFewH ? size - h0 : kFewH);
  float xv[kFewH][R], acc[kFewH][R];
#pragma unroll
  for (int h = 0; h < kFewH; ++h)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      xv[h][r] = h < hs && r < count ? to_f32(x[r * size + h0 + h]) : 0.0f;
      acc[h][r] = 0.0f;
    }
  for (int64_t c = (int64_t)threadIdx.x * VEC; c < classes; c += kFewThreads * VEC) {
    Pack<float, VEC> gv[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (r < count)
        gv[r] = load_pack<float, VEC>(g + r * ldg + c);
      else
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          gv[r].v[j] = 0.0f;
    Pack<T, VEC> wv[kFewH];
    if (dx)
#pragma unroll
      for (int h = 0; h < kFewH; ++h)
        if (h < hs)
          wv[h] = load_pack_stream<T, VEC>(w + (h0 + h) * classes + c);
#pragma unroll
    for (int h = 0; h < kFewH; ++h) {
      if (h >= hs)
        continue;
      if (dx)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            acc[h][r] = fmaf(gv[r].v[j], wv[h].f(j), acc[h][r]);
      if (dw) {
        T *to = dw + (h0 + h) * classes + c;
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          o[j] = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            o[j] = fmaf(xv[h][r], gv[r].v[j], o[j]);
        if (accum_dw) {
          const Pack<T, VEC> old = load_pack<T, VEC>(to);
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            o[j] += old.f(j);
        }
        store_pack<T, VEC>(to, o, keep);
      }
    }
  }
  if (!dx)
    return;
#pragma unroll
  for (int h = 0; h < kFewH; ++h)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float s = warp_sum(acc[h][r]);
      if (lane == 0)
        sums[warp][h * R + r] = s;
    }
  __syncthreads();
  if ((int)threadIdx.x < kFewH * R) {
    const int h = threadIdx.x / R, r = threadIdx.x % R;
    if (h < hs && r < count) {
      float s = 0.0f;
#pragma unroll
      for (int u = 0; u < kFewThreads / 32; ++u)
        s += sums[u][threadIdx.x];
      T *to = dx + r * size + h0 + h;
      *to = from_f32<T>(accum_dx ? s + to_f32(*to) : s);
    }
  }
}

template <typename T, int R, int VEC>
int few_logits(const T *x, const T *w, const T *bias, const LossRows &r, int count, int64_t size, float *g, int64_t ldg,
               cudaStream_t st) {
  constexpr int kCols = few_lanes<T, VEC>() * VEC;
  const dim3 grid((unsigned)((r.classes + kCols - 1) / kCols));
  constexpr int kXs = kFewValues * 4, kSums = kFewThreads / 32 * R * kCols * 4, kRing = VEC * sizeof(T) == 16 ? kFewRing : 0;
  constexpr int kMost = kRing + kXs > kSums ? kRing + kXs : kSums;
  const int smem = std::max(kRing + (int)std::min<int64_t>(kXs, size * R * 4), kSums);
  static std::atomic<bool> configured[64]{};
  int dev = 0;
  NB_CUDA(cudaGetDevice(&dev));
  if (!configured[dev & 63]) {
    NB_CUDA(cudaFuncSetAttribute(few_logits_kernel<T, R, VEC, Out::kGrad>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
    NB_CUDA(cudaFuncSetAttribute(few_logits_kernel<T, R, VEC, Out::kSums>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
    configured[dev & 63] = true;
  }
  if (g)
    NB_CUDA(launch_dependent(few_logits_kernel<T, R, VEC, Out::kGrad>, grid, dim3(kFewThreads), smem, st, x, w, bias, r,
                             count, size, g, ldg));
  else
    NB_CUDA(launch_dependent(few_logits_kernel<T, R, VEC, Out::kSums>, grid, dim3(kFewThreads), smem, st, x, w, bias, r,
                             count, size, g, ldg));
  return NB200_OK;
}

// f(rows rounded up to 1, 2, 4 or 8; values an access) as compile-time constants
template <typename T, typename F> int few_variant(int64_t rows, bool vec, F f) {
  auto with_vec = [&](auto r) -> int {
    return vec ? f(r, std::integral_constant<int, kPackOf<T>>{}) : f(r, std::integral_constant<int, 1>{});
  };
  return rows <= 1   ? with_vec(std::integral_constant<int, 1>{})
         : rows <= 2 ? with_vec(std::integral_constant<int, 2>{})
         : rows <= 4 ? with_vec(std::integral_constant<int, 4>{})
                     : with_vec(std::integral_constant<int, 8>{});
}

} // namespace nb200
