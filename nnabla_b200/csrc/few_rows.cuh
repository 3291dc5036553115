// The classifying head for up to eight rows: W decides, 2 or 4 bytes for every two to sixteen operations a row, so that the
// CUDA cores in fp32 keep up with HBM and nothing is laid out first.
#pragma once
#include "loss_gemm.cuh"

namespace nb200 {

constexpr int kFewRows = 8;
constexpr int kFewThreads = 256, kFewGradThreads = 256, kFewValues = 8192; // values: of x held in shared memory at a time
// Two fp32 multiply-adds in one instruction.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

template <int R> struct alignas(R > 1 ? 16 : 8) Few { // a value of x of each row, twice
  uint64_t v[R];
};

constexpr int kFewBatch = 4, kFewBatches = 3;                         // packs a batch of copies, batches on the way
constexpr int kFewRing = kFewBatch * kFewBatches * kFewThreads * 16; // bytes

constexpr int kFewLanes = 16; // that read a row of W side by side
// Classes of a group. kShift: the sixteen accesses of a row begin up to VEC - 1 values in front of the group's first class.
template <typename T, bool kShift> constexpr int few_columns() { return (kFewLanes - (kShift ? 1 : 0)) * kPackOf<T>; }
// Shared memory in front of x: the ring, or in its place the warps' sums (kShift: the half warps').
template <typename T, int R, bool kShift> constexpr int few_fixed_bytes() {
  const int sums = kFewThreads / (kShift ? kFewLanes : 32) * R * few_columns<T, kShift>() * 4;
  return kFewRing > sums ? kFewRing : sums;
}

// l = x W + b for a group of classes: half a warp reads 256 bytes of a row of W at a time ([1, 2048] . [2048,
// 32000] bf16, with the second kernel, 26.4 us; with runs of 128 bytes 30.2). Where the groups are fewer than the SMs a cluster
// of `splits` blocks shares one, each with its part of K, and its first block adds up their sums, in order (where they are
// enough that costs more than it brings: 29.6 us with two blocks, 33.7 with four). Of those kSums leaves the maximum and the
// sum of the exponentials, kGrad G in fp32.
// kShift: rows of W that begin anywhere. A thread's rows are sixteen apart, a multiple of VEC, so that all of them begin equally
// far behind a 16-byte boundary; it reads from the boundaries, and its sums are those of the classes `shift` further back.
// (Value by value, in runs of 128 or 64 bytes: [2, 4096] . [4096, 131071] fp32 1147 us, 323 with 131072 classes.)
template <typename T, int R, bool kShift, Out kOut>
__global__ void __launch_bounds__(kFewThreads) few_logits_kernel(const T *__restrict__ x, const T *__restrict__ w,
                                                                 const T *__restrict__ bias, LossRows rows, int count,
                                                                 int64_t size, int splits, float *__restrict__ g,
                                                                 int64_t ldg) {
  constexpr int VEC = kPackOf<T>, kCols = few_columns<T, kShift>(), kStep = kFewThreads / kFewLanes;
  constexpr int kWarps = kFewThreads / 32, kParts = kShift ? kStep : kWarps; // of the sums: one a half warp, or a warp
  static_assert(kStep % VEC == 0, "a thread's rows begin alike");
  constexpr int kFewK = kFewValues / R;
  extern __shared__ __align__(16) uint8_t few_smem[];
  uint4(*ring)[kFewThreads] = reinterpret_cast<uint4(*)[kFewThreads]>(few_smem); // [kFewBatches * kFewBatch]
  float(*sums)[R][kCols] = reinterpret_cast<float(*)[R][kCols]>(few_smem);       // behind the last use of the ring
  float *xs = reinterpret_cast<float *>(few_smem + few_fixed_bytes<T, R, kShift>());
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t group = blockIdx.x / splits;
  const int split = blockIdx.x - (int)group * splits;
  const int64_t each = (size + splits - 1) / splits, ka = split * each, kb = ka + each < size ? ka + each : size;
  const int k_first = threadIdx.x / kFewLanes;
  const int64_t classes = rows.classes, c0 = group * kCols;
  const int shift = kShift ? (int)(reinterpret_cast<uintptr_t>(w) / sizeof(T) + (ka + k_first) * classes) & (VEC - 1) : 0;
  const int64_t c = c0 + (threadIdx.x % kFewLanes) * VEC - shift; // of the thread's access
  const bool here = c < classes;                                  // (kShift: some of it; otherwise VEC divides classes)
  constexpr int kPairs = VEC / 2;                                 // of neighbouring classes
  uint64_t acc[R][kPairs];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < kPairs; ++j)
      acc[r][j] = 0;
  // W by asynchronous copies, each thread for itself: kFewBatches batches of kFewBatch packs on the way, whatever the compiler
  // makes of the registers (of eight ordinary loads a step it kept few in flight: 3.4 TB/s). The batches are those of the loop
  // below, a full piece of K being whole batches.
  static_assert(kFewK % (kFewBatch * kStep) == 0, "a piece of K is whole batches");
  int64_t next = ka + k_first;
  int fetched = 0, batch = 0;
  auto fetch = [&]() {
    const int at = fetched++ % kFewBatches * kFewBatch;
#pragma unroll
    for (int u = 0; u < kFewBatch; ++u, next += kStep)
      if (here && next < kb) {
        const int64_t e = next * classes + c; // (kShift: beside its row an access reads the neighbouring rows)
        if (!kShift || (e >= 0 && e + VEC <= size * classes)) {
          cp_async16(&ring[at + u][threadIdx.x], w + e);
        } else { // nothing in front of W or behind it
          Pack<T, VEC> p;
          p.clear();
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if (e + j >= 0 && e + j < size * classes)
              p.set(j, w[e + j]);
          *reinterpret_cast<Pack<T, VEC> *>(&ring[at + u][threadIdx.x]) = p;
        }
      }
    cp_async_commit();
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
      uint64_t wv[kPairs];
#pragma unroll
      for (int j = 0; j < kPairs; ++j)
        wv[j] = pair_of(v.f(2 * j), v.f(2 * j + 1));
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float xv = xs[k * R + r];
        const uint64_t xx = pair_of(xv, xv);
#pragma unroll
        for (int j = 0; j < kPairs; ++j)
          acc[r][j] = fma2(xx, wv[j], acc[r][j]);
      }
    };
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
  }
  cp_async_wait<0>();
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float2 both = unpair(acc[r][j / 2]);
      float s = j & 1 ? both.y : both.x;
      if constexpr (kShift) { // the halves of a warp begin differently
        const int i = lane % kFewLanes * VEC + j - shift;
        if (i >= 0 && i < kCols)
          sums[k_first][r][i] = s;
      } else {
        s += __shfl_xor_sync(0xffffffffu, s, kFewLanes);
        if (lane < kFewLanes)
          sums[warp][r][lane * VEC + j] = s;
      }
    }
  __syncthreads();
  float *own = &sums[0][0][0]; // [R][kCols], the block's
  for (int i = threadIdx.x; i < R * kCols; i += kFewThreads) {
    float s = 0.0f;
#pragma unroll
    for (int u = 0; u < kParts; ++u)
      s += own[u * R * kCols + i];
    own[i] = s;
  }
  if (splits > 1)
    cluster_barrier();
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
    cluster_barrier();
}

// dx = G W^T and dW = x^T G in one pass over W. A thread has eight columns of G in registers, [R][8] in fp32, and walks along
// the rows of W: of each it loads its columns, stores those of dW and has R products for dx, which its warp sums up (the first
// steps exchange halves of the values, so that the sixteen of two rows take sixteen shuffles). The sums of a block's columns, 256 * 8, go to
// partial[block column][R][size]. (With the threads along a row and G read from L2 for every four rows of W [5, 1792] . [1792,
// 109056] bf16 took 398 us.)
constexpr int kFewWalk = 32; // rows of W between two exchanges of the warps' sums
template <typename T, int R, int VEC>
__global__ void __launch_bounds__(kFewGradThreads) few_grads_kernel(const T *__restrict__ x, const T *__restrict__ w,
                                                                    const float *__restrict__ g, int64_t ldg, bool want_dx,
                                                                    T *dw, float *__restrict__ partial, int count,
                                                                    int64_t size, int64_t slab, int64_t classes,
                                                                    bool accum_dw, bool keep) {
  constexpr int kGroups = 8 / VEC, kWarps = kFewGradThreads / 32; // groups of VEC neighbouring columns
  __shared__ Few<R> xs[kFewWalk];
  __shared__ float sums[kWarps][kFewWalk][R];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c0 = (int64_t)blockIdx.x * kFewGradThreads * 8 + threadIdx.x * VEC;
  const int64_t h0 = blockIdx.y * slab, h1 = h0 + slab < size ? h0 + slab : size;
  auto column = [&](int i) { return c0 + (int64_t)i * kFewGradThreads * VEC; }; // of group i
  uint64_t gv[R][4];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float f[8];
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        f[i * VEC + j] = r < count && column(i) < classes ? g[r * ldg + column(i) + j] : 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      gv[r][j] = pair_of(f[2 * j], f[2 * j + 1]);
  }
  Pack<T, VEC> next[2][kGroups]; // the next two rows of W
  auto fetch = [&](int64_t h, int to) {
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
      if (want_dx && h < h1 && column(i) < classes)
        next[to][i] = load_pack_stream<T, VEC>(w + h * classes + column(i));
      else
        next[to][i].clear();
  };
  fetch(h0, 0);
  fetch(h0 + 1, 1);
  for (int64_t h = h0; h < h1; h += kFewWalk) {
    const int n = (int)(h1 - h < kFewWalk ? h1 - h : kFewWalk);
    for (int i = threadIdx.x; i < kFewWalk * R; i += kFewGradThreads) {
      const int r = i / kFewWalk, k = i % kFewWalk;
      const float v = r < count && k < n ? to_f32(x[r * size + h + k]) : 0.0f;
      xs[k].v[r] = pair_of(v, v);
    }
    __syncthreads();
    // two rows at a time, for the latency of their chains
    for (int k = 0; k < n; k += 2) {
      float s[2 * R];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint64_t wv[4];
        {
          float f[8];
#pragma unroll
          for (int i = 0; i < kGroups; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
              f[i * VEC + j] = next[q][i].f(j);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            wv[j] = pair_of(f[2 * j], f[2 * j + 1]);
        }
        fetch(h + k + q + 2, q);
        if (dw && k + q < n) {
          const Few<R> xv = xs[k + q];
          float o[kGroups][VEC];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint64_t t = 0;
#pragma unroll
            for (int r = 0; r < R; ++r)
              t = fma2(xv.v[r], gv[r][j], t);
            const float2 both = unpair(t);
            o[2 * j / VEC][2 * j % VEC] = both.x;
            o[(2 * j + 1) / VEC][(2 * j + 1) % VEC] = both.y;
          }
#pragma unroll
          for (int i = 0; i < kGroups; ++i) {
            if (column(i) >= classes)
              continue;
            T *to = dw + (h + k + q) * classes + column(i);
            if (accum_dw) {
              const Pack<T, VEC> old = load_pack<T, VEC>(to);
#pragma unroll
              for (int j = 0; j < VEC; ++j)
                o[i][j] += old.f(j);
            }
            store_pack<T, VEC>(to, o[i], keep);
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          uint64_t t = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            t = fma2(gv[r][j], wv[j], t);
          const float2 both = unpair(t);
          s[q * R + r] = both.x + both.y;
        }
      }
      if (want_dx) {
        int d = 16;
#pragma unroll
        for (int m = R; m >= 1; m /= 2, d /= 2) {
          const bool upper = lane & d;
#pragma unroll
          for (int i = 0; i < m; ++i) {
            const float away = upper ? s[i] : s[i + m];
            s[i] = (upper ? s[i + m] : s[i]) + __shfl_xor_sync(0xffffffffu, away, d);
          }
        }
#pragma unroll
        for (; d >= 1; d /= 2)
          s[0] += __shfl_xor_sync(0xffffffffu, s[0], d);
        const int i = lane / (16 / R); // lane's leading bits are the row of W and the row that it ended with
        if (lane % (16 / R) == 0 && k + i / R < n)
          sums[warp][k + i / R][i % R] = s[0];
      }
    }
    __syncthreads();
    if (want_dx)
      for (int i = threadIdx.x; i < kFewWalk * R; i += kFewGradThreads) {
        const int r = i / kFewWalk, k = i % kFewWalk;
        if (k >= n || r >= count)
          continue;
        float s = 0.0f;
#pragma unroll
        for (int u = 0; u < kWarps; ++u)
          s += sums[u][k][r];
        partial[((int64_t)blockIdx.x * count + r) * size + h + k] = s;
      }
  }
}

template <typename T, int R, bool kShift>
int few_logits(const T *x, const T *w, const T *bias, const LossRows &r, int count, int64_t size, float *g, int64_t ldg,
               cudaStream_t st) {
  constexpr int kCols = few_columns<T, kShift>(), kXs = kFewValues * 4, kFixed = few_fixed_bytes<T, R, kShift>();
  const int64_t groups = (r.classes + kCols - 1) / kCols;
  int splits = 1;
  while (splits < 8 && groups * splits < sm_count() && size >= 128 * splits)
    splits *= 2;
  const int smem = kFixed + (int)std::min<int64_t>(kXs, (size + splits - 1) / splits * R * 4);
  auto kernel = g ? few_logits_kernel<T, R, kShift, Out::kGrad> : few_logits_kernel<T, R, kShift, Out::kSums>;
  static std::atomic<bool> configured[64]{};
  int dev = 0;
  NB_CUDA(cudaGetDevice(&dev));
  if (!configured[dev & 63]) {
    NB_CUDA(cudaFuncSetAttribute(few_logits_kernel<T, R, kShift, Out::kGrad>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFixed + kXs));
    NB_CUDA(cudaFuncSetAttribute(few_logits_kernel<T, R, kShift, Out::kSums>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFixed + kXs));
    configured[dev & 63] = true;
  }
  NB_CUDA(launch_clusters(kernel, (unsigned)(groups * splits), splits, kFewThreads, smem, st, x, w, bias, r, count, size,
                          splits, g, ldg));
  return NB200_OK;
}

// f(rows rounded up to 1, 2, 4 or 8) as a compile-time constant
template <typename F> int few_variant(int64_t rows, F f) {
  return rows <= 1   ? f(std::integral_constant<int, 1>{})
         : rows <= 2 ? f(std::integral_constant<int, 2>{})
         : rows <= 4 ? f(std::integral_constant<int, 4>{})
                     : f(std::integral_constant<int, 8>{});
}
// Whether rows of W, or of dW, begin at 16-byte boundaries.
template <typename T> bool few_aligned(const T *w, int64_t classes) { return classes % kPackOf<T> == 0 && aligned16(w); }

} // namespace nb200
