// The classifying head for up to eight rows: W decides, 2 or 4 bytes for every two to sixteen operations a row, which the CUDA
// cores make in fp32 with nothing laid out first. The loss of one to four rows is near HBM (fp32 [2, 4096] . [4096, 131071] 340 us
// for 327 of bytes), of eight rows at 80 %; the gradients' pass at 70 to 95 % of it (907 and 694 us for 655).
#pragma once
#include "loss_gemm.cuh"

namespace nb200 {

constexpr int kFewRows = 8;
constexpr int kFewThreads = 256, kFewValues = 8192; // values: of x held in shared memory at a time
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

template <int R> struct alignas(R < 4 ? 4 * R : 16) Values { // a value of x of each row
  float v[R];
};
template <int R> struct alignas(R > 1 ? 16 : 8) Few { // a value of x of each row, twice
  uint64_t v[R];
};

constexpr int kFewBatch = 4, kFewBatches = 3;                         // packs a batch of copies, batches on the way
constexpr int kFewRing = kFewBatch * kFewBatches * kFewThreads * 16; // bytes

constexpr int kFewLanes = 16; // that read a row of W side by side
// Accesses of a thread in a row of W: two where that makes eight classes, of five to eight rows, for which one look at x serves.
template <typename T, int R> constexpr int few_packs() { return R == 8 && sizeof(T) == 4 ? 2 : 1; }
// Classes of a group. kShift: the accesses of a row begin up to VEC - 1 values in front of the group's first class.
template <typename T, int R, bool kShift> constexpr int few_columns() {
  return (kFewLanes * few_packs<T, R>() - (kShift ? 1 : 0)) * kPackOf<T>;
}
// Shared memory in front of x: the ring, or in its place the warps' sums (kShift: the half warps').
template <typename T, int R, bool kShift> constexpr int few_fixed_bytes() {
  const int sums = kFewThreads / (kShift ? kFewLanes : 32) * R * few_columns<T, R, kShift>() * 4;
  return kFewRing > sums ? kFewRing : sums;
}

// l = x W + b for a group of classes: half a warp reads 256 bytes of a row of W at a time ([1, 2048] . [2048,
// 32000] bf16, with the second kernel, 26.4 us; with runs of 128 bytes 30.2). Where the groups are fewer than the SMs a cluster
// of `splits` blocks shares one, each with its part of K, and its first block adds up their sums, in order (where they are
// enough that costs more than it brings: 29.6 us with two blocks, 33.7 with four). Of those kSums leaves the maximum and the
// sum of the exponentials, kGrad G in fp32.
// kShift: rows of W that begin anywhere. A thread's rows are sixteen apart, a multiple of VEC, so that all of them begin equally
// far behind a 16-byte boundary; it reads from the boundaries, and its sums are those of the classes `shift` further back.
// [2, 4096] . [4096, 131071] fp32 340 us, 323 with 131072 classes; 1147 value by value, in runs of 128 bytes. [8, 4096] fp32
// 400 and 323 us; 500 and 394 with a single access a thread, which looks at x twice as often.
template <typename T, int R, bool kShift, Out kOut>
__global__ void __launch_bounds__(kFewThreads) few_logits_kernel(const T *__restrict__ x, const T *__restrict__ w,
                                                                 const T *__restrict__ bias, LossRows rows, int count,
                                                                 int64_t size, int splits, float *__restrict__ g,
                                                                 int64_t ldg) {
  constexpr int VEC = kPackOf<T>, kCols = few_columns<T, R, kShift>(), kStep = kFewThreads / kFewLanes;
  constexpr int kPacks = few_packs<T, R>(), kRows = kFewBatch / kPacks; // of a row; rows of a batch
  constexpr int kWarps = kFewThreads / 32, kParts = kShift ? kStep : kWarps; // of the sums: one a half warp, or a warp
  static_assert(kStep % VEC == 0, "a thread's rows begin alike");
  constexpr int kFewK = kFewValues / R;
  extern __shared__ __align__(16) uint8_t few_smem[];
  uint4(*ring)[kFewThreads] = reinterpret_cast<uint4(*)[kFewThreads]>(few_smem); // [kFewBatches * kFewBatch]
  float(*sums)[R][kCols] = reinterpret_cast<float(*)[R][kCols]>(few_smem);       // behind the last use of the ring
  Values<R> *xs = reinterpret_cast<Values<R> *>(few_smem + few_fixed_bytes<T, R, kShift>());
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t group = blockIdx.x / splits;
  const int split = blockIdx.x - (int)group * splits;
  const int64_t each = (size + splits - 1) / splits, ka = split * each, kb = ka + each < size ? ka + each : size;
  const int k_first = threadIdx.x / kFewLanes;
  const int64_t classes = rows.classes, c0 = group * kCols;
  const int shift = kShift ? (int)(reinterpret_cast<uintptr_t>(w) / sizeof(T) + (ka + k_first) * classes) & (VEC - 1) : 0;
  const int64_t c = c0 + (threadIdx.x % kFewLanes) * VEC - shift; // of the thread's first access, the others kNext further on
  constexpr int kNext = kFewLanes * VEC, kPairs = VEC / 2;        // pairs of neighbouring classes
  auto here = [&](int p) { return c + p * kNext < classes; };     // (kShift: some of it; otherwise VEC divides classes)
  uint64_t acc[R][kPacks * kPairs];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < kPacks * kPairs; ++j)
      acc[r][j] = 0;
  // W by asynchronous copies, each thread for itself: kFewBatches batches of kFewBatch packs on the way, whatever the compiler
  // makes of the registers (of eight ordinary loads a step it kept few in flight: 3.4 TB/s). The batches are those of the loop
  // below, a full piece of K being whole batches.
  static_assert(kFewK % (kRows * kStep) == 0, "a piece of K is whole batches");
  int64_t next = ka + k_first, e = next * classes + c; // the next access's row and first value in W
  // kShift: beside its row an access reads the neighbouring rows, but nothing in front of W or behind it. e < whole, unsigned: an
  // access that lies in W.
  const int64_t all = size * classes, step = kStep * classes;
  const uint64_t whole = all < VEC ? 0 : (uint64_t)(all - VEC + 1);
  int fetched = 0, batch = 0;
  auto fetch = [&]() {
    const int at = fetched++ % kFewBatches * kFewBatch;
#pragma unroll
    for (int u = 0; u < kRows; ++u, next += kStep, e += step)
#pragma unroll
      for (int p = 0; p < kPacks; ++p)
        if (here(p) && next < kb) {
          const int64_t first = e + p * kNext;
          uint4 *to = &ring[at + u * kPacks + p][threadIdx.x];
          if (!kShift || (uint64_t)first < whole) {
            cp_async16(to, w + first);
          } else {
            Pack<T, VEC> some;
            some.clear();
#pragma unroll
            for (int j = 0; j < VEC; ++j)
              if (first + j >= 0 && first + j < all)
                some.set(j, w[first + j]);
            *reinterpret_cast<Pack<T, VEC> *>(to) = some;
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
    // (all rows' loads together, and several k's: with a row after the other a piece of K waited for eight round trips)
#pragma unroll(R == 1 ? 8 : R == 2 ? 4 : 2)
    for (int k = threadIdx.x; k < n; k += kFewThreads) {
      Values<R> v;
#pragma unroll
      for (int r = 0; r < R; ++r)
        v.v[r] = r < count ? to_f32(x[r * size + k0 + k]) : 0.0f;
      xs[k] = v;
    }
    __syncthreads();
    for (int k = k_first; k < n; k += kRows * kStep) {
      const int at = batch++ % kFewBatches * kFewBatch;
      cp_async_wait<kFewBatches - 1>();
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        if (!here(0) || k + u * kStep >= n)
          continue;
        const Values<R> xv = xs[k + u * kStep];
#pragma unroll
        for (int p = 0; p < kPacks; ++p) { // (of an access behind the last class there are no sums)
          const Pack<T, VEC> v = *reinterpret_cast<const Pack<T, VEC> *>(&ring[at + u * kPacks + p][threadIdx.x]);
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            const uint64_t wv = pair_of(v.f(2 * j), v.f(2 * j + 1));
#pragma unroll
            for (int r = 0; r < R; ++r)
              acc[r][p * kPairs + j] = fma2(pair_of(xv.v[r], xv.v[r]), wv, acc[r][p * kPairs + j]);
          }
        }
      }
      fetch();
    }
  }
  cp_async_wait<0>();
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < kPacks * VEC; ++j) {
      const float2 both = unpair(acc[r][j / 2]);
      float s = j & 1 ? both.y : both.x;
      const int i = lane % kFewLanes * VEC + j / VEC * kNext + j % VEC - shift;
      if constexpr (kShift) { // the halves of a warp begin differently
        if (i >= 0 && i < kCols)
          sums[k_first][r][i] = s;
      } else {
        s += __shfl_xor_sync(0xffffffffu, s, kFewLanes);
        if (lane < kFewLanes)
          sums[warp][r][i] = s;
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
// steps exchange halves of the values, so that the sixteen of two rows take sixteen shuffles). The sums of a block's columns,
// kFewBlock, go to partial[block column][R][size]. (With the threads along a row and G read from L2 for every four rows of W
// [5, 1792] . [1792, 109056] bf16 took 398 us.)
// kShift: rows of W that begin anywhere. A block's rows are VEC apart, so that all of them begin `shift` values behind a 16-byte
// boundary, and its columns begin `shift` further back; a row's two ends, fewer than VEC values each, are the last block
// column's. (All of it value by value: [8, 4096] . [4096, 131071] fp32 1032 us, 907 so; bytes 655.)
// Bound by latency with 64 bytes of W ahead a thread: two blocks an SM with their registers, of one or two rows three
// ([8, 4096] . [4096, 131072] fp32 1188 us with one block, 891 with two; [1, 2048] . [2048, 100000] 279 with two, 255 with three).
template <typename T, int R, bool kShift>
__global__ void __launch_bounds__(kFewGradThreads, R >= 4 ? 2 : 3) few_grads_kernel(const T *__restrict__ x, const T *__restrict__ w,
                                                                    const float *__restrict__ g, int64_t ldg, bool want_dx,
                                                                    T *dw, float *__restrict__ partial, int count,
                                                                    int64_t size, int64_t slab, int64_t classes,
                                                                    bool accum_dw, bool keep) {
  constexpr int VEC = kPackOf<T>, kGroups = 8 / VEC, kWarps = kFewGradThreads / 32; // groups of VEC neighbouring columns
  constexpr int kStep = kShift ? VEC : 1;                                           // rows of W from one of the block's to the next
  __shared__ Few<R> xs[kFewWalk];
  __shared__ float sums[kWarps][kFewWalk][R];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = kShift ? (int)(blockIdx.y % kStep) : 0;
  const uintptr_t begin = reinterpret_cast<uintptr_t>(want_dx ? w : dw) / sizeof(T); // (W and dW, where both: equally far)
  const int shift = kShift ? (int)(begin + first * classes) & (VEC - 1) : 0;
  const int64_t c0 = (int64_t)blockIdx.x * kFewBlock + threadIdx.x * VEC - shift;
  // the block's rows are first + i kStep, i in [i0, i1)
  const int64_t mine = (size - first + kStep - 1) / kStep, i0 = blockIdx.y / kStep * slab, i1 = i0 + slab < mine ? i0 + slab : mine;
  auto row = [&](int64_t i) { return first + i * kStep; };
  if constexpr (kShift)
    if (blockIdx.x == gridDim.x - 1) { // a row's ends: in front of the first access that lies in it, and behind the last
      const int64_t left = shift == 0 ? 0 : VEC - shift < classes ? VEC - shift : classes;
      const int64_t last = (classes + shift) / VEC * VEC - shift, right = last > left ? last : left;
      for (int64_t i = i0 + threadIdx.x; i < i1; i += kFewGradThreads) {
        float s[R];
#pragma unroll
        for (int r = 0; r < R; ++r)
          s[r] = 0.0f;
        for (int64_t c = left > 0 ? 0 : right; c < classes; c = c + 1 == left ? right : c + 1) {
          const int64_t at = row(i) * classes + c;
          const float wv = want_dx ? to_f32(w[at]) : 0.0f;
          float o = 0.0f;
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (r < count) {
              const float f = g[r * ldg + c];
              s[r] = fmaf(f, wv, s[r]);
              o = fmaf(to_f32(x[r * size + row(i)]), f, o);
            }
          if (dw)
            dw[at] = from_f32<T>(accum_dw ? o + to_f32(dw[at]) : o);
        }
        if (want_dx)
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (r < count)
              partial[((int64_t)blockIdx.x * count + r) * size + row(i)] = s[r];
      }
      return;
    }
  auto column = [&](int i) { return c0 + (int64_t)i * kFewGradThreads * VEC; }; // of group i
  auto full = [&](int i) { return kShift ? column(i) >= 0 && column(i) + VEC <= classes : column(i) < classes; };
  uint64_t gv[R][4];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float f[8];
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        f[i * VEC + j] = r < count && full(i) ? g[r * ldg + column(i) + j] : 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      gv[r][j] = pair_of(f[2 * j], f[2 * j + 1]);
  }
  Pack<T, VEC> next[2][kGroups]; // the next two rows of W
  auto fetch = [&](int64_t i, int to) {
#pragma unroll
    for (int u = 0; u < kGroups; ++u)
      if (want_dx && i < i1 && full(u))
        next[to][u] = load_pack_stream<T, VEC>(w + row(i) * classes + column(u));
      else
        next[to][u].clear();
  };
  fetch(i0, 0);
  fetch(i0 + 1, 1);
  for (int64_t i = i0; i < i1; i += kFewWalk) {
    const int n = (int)(i1 - i < kFewWalk ? i1 - i : kFewWalk);
    for (int t = threadIdx.x; t < kFewWalk * R; t += kFewGradThreads) {
      const int r = t / kFewWalk, k = t % kFewWalk;
      const float v = r < count && k < n ? to_f32(x[r * size + row(i + k)]) : 0.0f;
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
          for (int u = 0; u < kGroups; ++u)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
              f[u * VEC + j] = next[q][u].f(j);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            wv[j] = pair_of(f[2 * j], f[2 * j + 1]);
        }
        fetch(i + k + q + 2, q);
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
          for (int u = 0; u < kGroups; ++u) {
            if (!full(u))
              continue;
            T *to = dw + row(i + k + q) * classes + column(u);
            if (accum_dw) {
              const Pack<T, VEC> old = load_pack<T, VEC>(to);
#pragma unroll
              for (int j = 0; j < VEC; ++j)
                o[u][j] += old.f(j);
            }
            store_pack<T, VEC>(to, o[u], keep);
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
          for (int t = 0; t < m; ++t) {
            const float away = upper ? s[t] : s[t + m];
            s[t] = (upper ? s[t + m] : s[t]) + __shfl_xor_sync(0xffffffffu, away, d);
          }
        }
#pragma unroll
        for (; d >= 1; d /= 2)
          s[0] += __shfl_xor_sync(0xffffffffu, s[0], d);
        const int t = lane / (16 / R); // lane's leading bits are the row of W and the row that it ended with
        if (lane % (16 / R) == 0 && k + t / R < n)
          sums[warp][k + t / R][t % R] = s[0];
      }
    }
    __syncthreads();
    if (want_dx)
      for (int t = threadIdx.x; t < kFewWalk * R; t += kFewGradThreads) {
        const int r = t / kFewWalk, k = t % kFewWalk;
        if (k >= n || r >= count)
          continue;
        float s = 0.0f;
#pragma unroll
        for (int u = 0; u < kWarps; ++u)
          s += sums[u][k][r];
        partial[((int64_t)blockIdx.x * count + r) * size + row(i + k)] = s;
      }
  }
}

template <typename T, int R, bool kShift>
int few_logits(const T *x, const T *w, const T *bias, const LossRows &r, int count, int64_t size, float *g, int64_t ldg,
               cudaStream_t st) {
  constexpr int kCols = few_columns<T, R, kShift>(), kXs = kFewValues * 4, kFixed = few_fixed_bytes<T, R, kShift>();
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
