// The classifying head for up to eight rows: W decides, 2 or 4 bytes for every two to sixteen operations a row, so that the
// CUDA cores in fp32 keep up with HBM and nothing is laid out first.
#pragma once
#include "loss_gemm.cuh"

namespace nb200 {

constexpr int kFewRows = 8;
constexpr int kFewThreads = 256, kFewGradThreads = 256, kFewValues = 8192; // values: of x held in shared memory at a time
constexpr int kFewBatch = 4, kFewBatches = 3;                         // packs a batch of copies, batches on the way
constexpr int kFewRing = kFewBatch * kFewBatches * kFewThreads * 16; // bytes

__device__ __forceinline__ void cp_async16(void *to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ptx::smem_u32(to)), "l"(from) : "memory");
}
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T, int VEC> constexpr int few_lanes() { return VEC * sizeof(T) == 16 ? 16 : 32; }
// Shared memory in front of x: the ring, or in its place the warps' sums.
template <typename T, int R, int VEC> constexpr int few_fixed_bytes() {
  const int ring = VEC * sizeof(T) == 16 ? kFewRing : 0, sums = kFewThreads / 32 * R * few_lanes<T, VEC>() * VEC * 4;
  return ring > sums ? ring : sums;
}

// l = x W + b for a group of classes, kLanes * VEC: half a warp reads 256 bytes of a row of W at a time ([1, 2048] . [2048,
// 32000] bf16, with the second kernel, 26.4 us; with runs of 128 bytes 30.2). Where the groups are fewer than the SMs a cluster
// of `splits` blocks shares one, each with its part of K, and its first block adds up their sums, in order (where they are
// enough that costs more than it brings: 29.6 us with two blocks, 33.7 with four). Of those kSums leaves the maximum and the
// sum of the exponentials, kGrad G in fp32.
template <typename T, int R, int VEC, Out kOut>
__global__ void __launch_bounds__(kFewThreads) few_logits_kernel(const T *__restrict__ x, const T *__restrict__ w,
                                                                 const T *__restrict__ bias, LossRows rows, int count,
                                                                 int64_t size, int splits, float *__restrict__ g,
                                                                 int64_t ldg) {
  constexpr bool kAsync = VEC * sizeof(T) == 16;
  constexpr int kLanes = few_lanes<T, VEC>(), kCols = kLanes * VEC, kWarps = kFewThreads / 32, kStep = kFewThreads / kLanes;
  constexpr int kFewK = kFewValues / R;
  extern __shared__ __align__(16) uint8_t few_smem[];
  uint4(*ring)[kFewThreads] = reinterpret_cast<uint4(*)[kFewThreads]>(few_smem); // [kFewBatches * kFewBatch]
  float(*sums)[R][kCols] = reinterpret_cast<float(*)[R][kCols]>(few_smem);       // behind the last use of the ring
  float *xs = reinterpret_cast<float *>(few_smem + few_fixed_bytes<T, R, VEC>());
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t group = blockIdx.x / splits;
  const int split = blockIdx.x - (int)group * splits;
  const int64_t classes = rows.classes, c0 = group * kCols, c = c0 + (threadIdx.x % kLanes) * VEC;
  const bool here = c < classes; // (VEC divides classes, or is 1)
  const int64_t each = (size + splits - 1) / splits, ka = split * each, kb = ka + each < size ? ka + each : size;
  float acc[R][VEC];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      acc[r][j] = 0.0f;
  // W by asynchronous copies, each thread for itself: kFewBatches batches of kFewBatch packs on the way, whatever the compiler
  // makes of the registers (of eight ordinary loads a step it kept few in flight: 3.4 TB/s). The batches are those of the loop
  // below, a full piece of K being whole batches.
  static_assert(!kAsync || kFewK % (kFewBatch * kStep) == 0, "a piece of K is whole batches");
  const int k_first = threadIdx.x / kLanes;
  int64_t next = ka + k_first;
  int fetched = 0, batch = 0;
  auto fetch = [&]() {
    if constexpr (kAsync) {
      const int at = fetched++ % kFewBatches * kFewBatch;
#pragma unroll
      for (int u = 0; u < kFewBatch; ++u, next += kStep)
        if (here && next < kb)
          cp_async16(&ring[at + u][threadIdx.x], w + next * classes + c);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  for (int i = 0; i < kFewBatches; ++i)
    fetch();
  for (int64_t k0 = ka; k0 < kb; k0 += kFewK) {
    const int n = (int)(kb - k0 < kFewK ? kb - k0 : kFewK);
    if (k0 > ka)
      __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll 4
      for (int k = threadIdx.x; k < n; k += kFewThreads)
        xs[k * R + r] = r < count ? to_f32(x[r * size + k0 + k]) : 0.0f;
    __syncthreads();
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
      for (int k = k_first; k < n; k += kFewBatch * kStep) {
        const int at = batch++ % kFewBatches * kFewBatch;
        cp_async_wait<kFewBatches - 1>();
        if (here)
#pragma unroll
          for (int u = 0; u < kFewBatch; ++u)
            if (k + u * kStep < n)
              add(*reinterpret_cast<const Pack<T, VEC> *>(&ring[at + u][threadIdx.x]), k + u * kStep);
        fetch();
      }
    } else if (here) {
#pragma unroll 8
      for (int k = k_first; k < n; k += kStep)
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
  float *own = &sums[0][0][0]; // [R][kCols], the block's
  for (int i = threadIdx.x; i < R * kCols; i += kFewThreads) {
    float s = 0.0f;
#pragma unroll
    for (int u = 0; u < kWarps; ++u)
      s += own[u * R * kCols + i];
    own[i] = s;
  }
  if (splits > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else
    __syncthreads();
  if (split == 0)
    for (int r = warp; r < count; r += kWarps) { // a warp a row
      const int64_t label = rows.label_of(r);
      MaxSum t{-INFINITY, 0.0f};
      for (int i = lane; i < kCols; i += 32) {
        if (c0 + i >= classes)
          continue;
        float l = own[r * kCols + i];
        for (int o = 1; o < splits; ++o) {
          uint32_t theirs;
          float f;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(theirs) : "r"(ptx::smem_u32(own + r * kCols + i)), "r"(o));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(theirs) : "memory");
          l += f;
        }
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
          rows.partial[(int64_t)r * rows.tiles + group] = make_float2(t.m, t.s);
      }
    }
  if (splits > 1) // no block leaves while the first may still read its sums
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// dx = G W^T and dW = x^T G in one pass over W: a block has kFewH rows of W, its threads walk along the classes. A pack of
// G, [R][VEC] in fp32 from L2, serves all of the block's rows.
constexpr int kFewH = 4;
template <typename T, int R, int VEC>
__global__ void __launch_bounds__(kFewGradThreads) few_grads_kernel(const T *__restrict__ x, const T *__restrict__ w,
                                                                const float *__restrict__ g, int64_t ldg, T *dx, T *dw,
                                                                int count, int64_t size, int64_t classes, bool accum_dx,
                                                                bool accum_dw, bool keep) {
  __shared__ float sums[kFewGradThreads / 32][kFewH * R];
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
  for (int64_t c = (int64_t)threadIdx.x * VEC; c < classes; c += kFewGradThreads * VEC) {
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
      for (int u = 0; u < kFewGradThreads / 32; ++u)
        s += sums[u][threadIdx.x];
      T *to = dx + r * size + h0 + h;
      *to = from_f32<T>(accum_dx ? s + to_f32(*to) : s);
    }
  }
}

template <typename T, int R, int VEC>
int few_logits(const T *x, const T *w, const T *bias, const LossRows &r, int count, int64_t size, float *g, int64_t ldg,
               cudaStream_t st) {
  constexpr int kCols = few_lanes<T, VEC>() * VEC, kXs = kFewValues * 4, kFixed = few_fixed_bytes<T, R, VEC>();
  const int64_t groups = (r.classes + kCols - 1) / kCols;
  int splits = 1;
  while (splits < 8 && groups * splits < sm_count() && size >= 128 * splits)
    splits *= 2;
  const int smem = kFixed + (int)std::min<int64_t>(kXs, (size + splits - 1) / splits * R * 4);
  auto kernel = g ? few_logits_kernel<T, R, VEC, Out::kGrad> : few_logits_kernel<T, R, VEC, Out::kSums>;
  static std::atomic<bool> configured[64]{};
  int dev = 0;
  NB_CUDA(cudaGetDevice(&dev));
  if (!configured[dev & 63]) {
    NB_CUDA(cudaFuncSetAttribute(few_logits_kernel<T, R, VEC, Out::kGrad>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFixed + kXs));
    NB_CUDA(cudaFuncSetAttribute(few_logits_kernel<T, R, VEC, Out::kSums>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFixed + kXs));
    configured[dev & 63] = true;
  }
  NB_CUDA(launch_clusters(kernel, (unsigned)(groups * splits), splits, kFewThreads, smem, st, x, w, bias, r, count, size,
                          splits, g, ldg));
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
