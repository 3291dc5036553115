// LayerNormalization over the trailing axes, forward and backward, in fp32, bf16 or fp16.
//
//   mean = sum x / C, variance = sum (x - mean)^2 / C, r = 1 / sqrt(variance + eps), u = (x - mean) r
//   y = u gamma + beta
//   g = dy gamma:  dx = r (g - mean(g) - u mean(g u));  dgamma = sum over rows of dy u, dbeta = sum over rows of dy
//
// HBM bound: a row is read once into registers (a warp's, for short rows, a block's, or a cluster's), the variance is taken from
// the centred values there, so that a large mean costs no digits. Measured, bf16: forward of [16384, 4096] 52 us (5.1 TB/s; its
// bytes 41), forward and gradients of [8192, 2048] 56 us (their bytes 26).
#include <algorithm>

#include "pdl.cuh"
#include "typed.cuh"

namespace nb200 {
namespace {

constexpr int kNormMaxWarps = 32;

// Sums of N (1 or 2) values over the threads of a row: a warp's, or (row_warps > 1, a multiple of 4) the block's. Every thread
// gets them. Two values share their shuffles: after the first step each half of the warp goes on with one of them. `turn`
// alternates the shared slots, so that one barrier a sum is enough.
template <int N>
__device__ __forceinline__ void row_sums(float (&v)[N], int row_warps, float (*slots)[N][kNormMaxWarps], int &turn) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (row_warps == 1) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = warp_sum(v[i]);
    return;
  }
  float s;
  if constexpr (N == 2) {
    const bool upper = lane >= 16;
    s = (upper ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, upper ? v[0] : v[1], 16);
  } else {
    s = v[0] + __shfl_xor_sync(0xffffffffu, v[0], 16);
  }
#pragma unroll
  for (int d = 8; d; d >>= 1)
    s += __shfl_xor_sync(0xffffffffu, s, d);
  float(*to)[kNormMaxWarps] = slots[turn];
  turn ^= 1;
  if (lane == 0)
    to[0][warp] = s;
  if (N == 2 && lane == 16)
    to[N - 1][warp] = s;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = 0.0f;
    for (int w = 0; w < row_warps; w += 4) {
      const float4 f = *reinterpret_cast<const float4 *>(&to[i][w]);
      v[i] += (f.x + f.y) + (f.z + f.w);
    }
  }
}

// Sums over the blocks of a cluster: each leaves its own in its shared memory and reads the others'. Fixed order.
template <int N> __device__ __forceinline__ void cluster_sums(float (&v)[N], float *slot, int blocks) {
  // (all threads hold the block's sums; slot: N floats of shared memory, not used again before the next cluster barrier)
  if (threadIdx.x == 0)
#pragma unroll
    for (int i = 0; i < N; ++i)
      slot[i] = v[i];
  cluster_barrier();
  // every warp for itself, a lane a block
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float f = 0.0f;
    if (lane < blocks) {
      const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(slot + i));
      uint32_t theirs;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(theirs) : "r"(mine), "r"(lane));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(theirs) : "memory");
    }
    v[i] = warp_sum(f);
  }
}

// A thread's part of a row: NV accesses of VEC values, a warp's side by side, so that their offsets are constants. kShift: the
// row begins `shift` values behind a 16-byte boundary (sizes that are no multiple of VEC), and the accesses lie on the
// boundaries; those across the row's ends go value by value. Column of access i: first + i * kStep.
template <int VEC, bool kShift> struct Columns {
  static constexpr int kStep = 32 * VEC;
  int first, end; // of the row (or the block's slice of it): [begin, end)
  int begin;
  __device__ __forceinline__ int at(int i) const { return first + i * kStep; }
  __device__ __forceinline__ bool full(int i) const {
    return kShift ? at(i) >= begin && at(i) + VEC <= end : at(i) < end;
  }
  __device__ __forceinline__ bool some(int i) const { return kShift ? at(i) + VEC > begin && at(i) < end : at(i) < end; }
  __device__ __forceinline__ bool has(int i, int j) const { return !kShift || (at(i) + j >= begin && at(i) + j < end); }
  // `mine` below: the row, or the parameters, plus `first`, so that the accesses have constant offsets from one address.
  // values that the row does not have: 0
  template <typename T, bool kStream> __device__ __forceinline__ Pack<T, VEC> load(const T *mine, int i) const {
    Pack<T, VEC> p;
    if (full(i)) {
      if constexpr (kStream)
        p = load_pack_stream<T, VEC>(mine + i * kStep);
      else
        p = load_pack<T, VEC>(mine + i * kStep);
    } else {
      p.clear();
      if (kShift && some(i))
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (has(i, j))
            p.set(j, mine[i * kStep + j]);
    }
    return p;
  }
  // of a parameter, whose columns are not aligned with the row's where kShift
  template <typename P> __device__ __forceinline__ Pack<P, VEC> parameter(const P *mine, int i, bool given, float none) const {
    Pack<P, VEC> p;
    if (!given) {
      p.fill(none); // (once, not chosen at every value)
    } else if constexpr (!kShift) {
      if (full(i))
        p = load_pack<P, VEC>(mine + i * kStep);
      else
        p.clear();
    } else {
      p.clear();
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (has(i, j))
          p.set(j, mine[i * kStep + j]);
    }
    return p;
  }
  template <typename T> __device__ __forceinline__ void store(T *mine, int i, const float (&v)[VEC], bool keep) const {
    if (full(i)) {
      store_pack<T, VEC>(mine + i * kStep, v, keep);
    } else if (kShift && some(i)) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (has(i, j))
          mine[i * kStep + j] = from_f32<T>(v[j]);
    }
  }
};
// The columns of this thread in a row that begins `shift` values behind a boundary; rank: of a cluster's blocks, slice of it.
template <int VEC, int NV, bool kShift>
__device__ __forceinline__ Columns<VEC, kShift> columns_of(int warp, int lane, int size, int shift, int rank, int slice) {
  Columns<VEC, kShift> c;
  const int from = rank * slice - (kShift ? shift : 0); // in front of the row for the first block
  c.first = from + warp * (NV * 32 * VEC) + lane * VEC;
  c.begin = from > 0 ? from : 0;
  c.end = size - from < slice ? size : from + slice;
  return c;
}
template <int VEC> __device__ __forceinline__ int shift_of(int64_t row, int size) { return (int)(row * size) & (VEC - 1); }

// Bound by HBM and by instruction issue (71 % of the slots at [16384, 4096] bf16: 18 instructions a value, and some 120 a warp and
// row for the two sums, hence four accesses a thread rather than more threads: 80 us with two, 52 with four).
// A row belongs to row_warps warps: a block holds one row, or (row_warps == 1) a row a warp, or (kCluster) a slice of a row; ROWS
// such rows at once, for which one barrier serves and one look at the parameters.
template <typename T, typename P, int VEC, int NV, int ROWS, bool kShift, bool kCluster>
__global__ void __launch_bounds__(512, 2) layer_norm_kernel(const T *__restrict__ x, const P *__restrict__ beta,
                                                         const P *__restrict__ gamma, T *y, float *__restrict__ mean_out,
                                                         float *__restrict__ var_out, int64_t rows, int size, float inv_size,
                                                         float eps, int row_warps, int cluster, int slice, bool keep) {
  static_assert(ROWS == 1 || !(kShift || kCluster), "rows of one block begin alike");
  __shared__ alignas(16) float slots[2][ROWS][kNormMaxWarps];
  __shared__ float shared_sums[2][1];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t block = kCluster ? blockIdx.x / cluster : blockIdx.x;
  const int64_t row = (row_warps == 1 ? block * (blockDim.x >> 5) + warp : block) * ROWS;
  if (row >= rows) // (whole warps, and never where the block shares a row)
    return;
  const int here = rows - row < ROWS ? (int)(rows - row) : ROWS;
  const auto cols = columns_of<VEC, NV, kShift>(row_warps == 1 ? 0 : warp, lane, size, shift_of<VEC>(row, size),
                                                kCluster ? (int)(blockIdx.x - block * cluster) : 0, kCluster ? slice : size + VEC);
  float v[ROWS][NV][VEC];
  {
    Pack<T, VEC> p[ROWS][NV];
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (q < here)
          p[q][i] = cols.template load<T, true>(x + (row + q) * size + cols.first, i);
        else
          p[q][i].clear();
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          v[q][i][j] = p[q][i].f(j);
  }
  int turn = 0;
  float mean[ROWS], r[ROWS];
#pragma unroll
  for (int q = 0; q < ROWS; ++q) {
    mean[q] = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        mean[q] += v[q][i][j];
  }
  row_sums<ROWS>(mean, row_warps, slots, turn);
  if constexpr (kCluster)
    cluster_sums<1>(mean, shared_sums[0], cluster);
#pragma unroll
  for (int q = 0; q < ROWS; ++q) {
    mean[q] *= inv_size;
    r[q] = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float m = cols.full(i) ? mean[q] : 0.0f;
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        v[q][i][j] -= m;
      if (kShift && !cols.full(i) && cols.some(i))
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          v[q][i][j] -= cols.has(i, j) ? mean[q] : 0.0f;
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        r[q] = fmaf(v[q][i][j], v[q][i][j], r[q]);
    }
  }
  row_sums<ROWS>(r, row_warps, slots, turn);
  if constexpr (kCluster)
    cluster_sums<1>(r, shared_sums[1], cluster);
  const bool first = kCluster ? threadIdx.x == 0 && blockIdx.x == block * cluster : row_warps == 1 ? lane == 0 : threadIdx.x == 0;
#pragma unroll
  for (int q = 0; q < ROWS; ++q) {
    const float var = r[q] * inv_size;
    r[q] = rsqrtf(var + eps);
    if (first && q < here) {
      if (mean_out)
        mean_out[row + q] = mean[q];
      if (var_out)
        var_out[row + q] = var;
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (!cols.some(i))
      continue;
    const Pack<P, VEC> g = cols.template parameter<P>(gamma + cols.first, i, gamma != nullptr, 1.0f);
    const Pack<P, VEC> b = cols.template parameter<P>(beta + cols.first, i, beta != nullptr, 0.0f);
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      if (q >= here)
        continue;
      float o[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        o[j] = fmaf(v[q][i][j] * r[q], g.f(j), b.f(j));
      cols.store(y + (row + q) * size + cols.first, i, o, keep);
    }
  }
  if constexpr (kCluster) // no block leaves while another may still read its sums
    cluster_barrier();
}

constexpr int kLongThreads = 512, kLongBlocks = 8;

// Rows that no cluster of the kernels around holds in registers: a cluster of eight blocks a row, each with an eighth of it,
// which it reads three times (from the second time on mostly from L2; [4, 200000] bf16 25 us, latency). kBackward: dx instead of y, with dy, mean and
// variance given.
template <typename T, typename P, bool kBackward>
__global__ void __cluster_dims__(kLongBlocks, 1, 1) __launch_bounds__(kLongThreads)
    layer_norm_long_kernel(const T *__restrict__ x, const T *__restrict__ dy, const P *__restrict__ beta,
                           const P *__restrict__ gamma, T *y, float *mean_io, float *var_io, int64_t size, float eps,
                           bool accum) {
  __shared__ alignas(16) float slots[2][kBackward ? 2 : 1][kNormMaxWarps];
  __shared__ float shared_sums[2][2];
  pdl_wait();
  pdl_trigger();
  const int64_t row = blockIdx.x / kLongBlocks;
  const int part = blockIdx.x % kLongBlocks;
  const int64_t each = (size + kLongBlocks - 1) / kLongBlocks, c0 = part * each;
  const int64_t c1 = c0 + each < size ? c0 + each : size;
  const T *xr = x + row * size;
  T *yr = y + row * size;
  const double inv = 1.0 / (double)size;
  int turn = 0;
  // f(c, sums) for this thread's values, 64 at a time in fp32 and those sums in 64 bits
  auto sum_up = [&](auto &s, auto f) {
    constexpr int kN = sizeof(s) / sizeof(float);
    double total[kN] = {};
    for (int64_t base = c0 + threadIdx.x; base < c1; base += 64 * kLongThreads) {
#pragma unroll
      for (int i = 0; i < kN; ++i)
        s[i] = 0.0f;
#pragma unroll 8
      for (int k = 0; k < 64; ++k)
        if (base + k * kLongThreads < c1)
          f(base + k * kLongThreads);
#pragma unroll
      for (int i = 0; i < kN; ++i)
        total[i] += s[i];
    }
#pragma unroll
    for (int i = 0; i < kN; ++i)
      s[i] = (float)total[i];
  };
  if constexpr (!kBackward) {
    float s[1];
    sum_up(s, [&](int64_t c) { s[0] += to_f32(xr[c]); });
    row_sums<1>(s, kLongThreads / 32, slots, turn);
    cluster_sums<1>(s, shared_sums[0], kLongBlocks);
    const float mean = (float)(s[0] * inv);
    sum_up(s, [&](int64_t c) {
      const float d = to_f32(xr[c]) - mean;
      s[0] = fmaf(d, d, s[0]);
    });
    row_sums<1>(s, kLongThreads / 32, slots, turn);
    cluster_sums<1>(s, shared_sums[1], kLongBlocks);
    const float var = (float)(s[0] * inv), r = rsqrtf(var + eps);
    if (part == 0 && threadIdx.x == 0) {
      if (mean_io)
        mean_io[row] = mean;
      if (var_io)
        var_io[row] = var;
    }
#pragma unroll 8
    for (int64_t c = c0 + threadIdx.x; c < c1; c += kLongThreads) {
      float o = (to_f32(xr[c]) - mean) * r;
      if (gamma)
        o *= to_f32(gamma[c]);
      if (beta)
        o += to_f32(beta[c]);
      yr[c] = from_f32<T>(o);
    }
  } else {
    const T *dr = dy + row * size;
    const float mean = mean_io[row], r = rsqrtf(var_io[row] + eps);
    float s[2];
    sum_up(s, [&](int64_t c) {
      const float g = gamma ? to_f32(dr[c]) * to_f32(gamma[c]) : to_f32(dr[c]);
      s[0] += g;
      s[1] = fmaf(g, (to_f32(xr[c]) - mean) * r, s[1]);
    });
    row_sums<2>(s, kLongThreads / 32, slots, turn);
    cluster_sums<2>(s, shared_sums[0], kLongBlocks);
    const float m1 = (float)(s[0] * inv), m2 = (float)(s[1] * inv);
#pragma unroll 8
    for (int64_t c = c0 + threadIdx.x; c < c1; c += kLongThreads) {
      const float g = gamma ? to_f32(dr[c]) * to_f32(gamma[c]) : to_f32(dr[c]);
      float o = r * (g - m1 - (to_f32(xr[c]) - mean) * r * m2);
      if (accum)
        o += to_f32(yr[c]);
      yr[c] = from_f32<T>(o);
    }
  }
  // no block leaves while another may still read its sums
  cluster_barrier();
}

// dx, and where kParams the sums over this block's rows of dy and dy u, each thread for the columns that it holds: a block (or
// a warp of it, for short rows) walks over the rows, and leaves partial sums [blocks][2][size] for layer_norm_param_kernel.
// kShift: the rows that a block walks over are VEC or a multiple of it apart, so that all begin alike. kCluster, for rows that
// one block does not hold: a cluster of blocks, each with a slice of the columns, takes one row (dx only).
// The next row of x and dy is on its way in registers while one is worked on (three rows in asynchronous copies to shared memory
// take no less: a row costs a warp some 200 instructions beside those of its values, with 16 warps an SM, and that is what bounds
// it: [8192, 2048] bf16 33 us, its bytes 15; half as many values a thread and twice the warps 43).
template <typename T, typename P, int VEC, int NV, bool kParams, bool kShift, bool kCluster>
__global__ void __launch_bounds__(512) layer_norm_backward_kernel(
    const T *__restrict__ x, const T *__restrict__ dy, const P *__restrict__ gamma, const float *__restrict__ mean,
    const float *__restrict__ var, T *dx, float *__restrict__ partial, int64_t rows, int size, float inv_size, float eps,
    int row_warps, int cluster, int slice, bool accum, bool keep) {
  __shared__ alignas(16) float slots[2][2][kNormMaxWarps];
  __shared__ float shared_sums[2][2];
  extern __shared__ float combine[]; // [warps][2][size], where a row is a warp's
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int64_t block = kCluster ? blockIdx.x / cluster : blockIdx.x, blocks = kCluster ? gridDim.x / cluster : gridDim.x;
  const int64_t first = row_warps == 1 ? block * warps + warp : block, stride = row_warps == 1 ? blocks * warps : blocks;
  const auto cols = columns_of<VEC, NV, kShift>(row_warps == 1 ? 0 : warp, lane, size, shift_of<VEC>(first, size),
                                                kCluster ? (int)(blockIdx.x - block * cluster) : 0, kCluster ? slice : size + VEC);
  float sum_dy[NV * VEC], sum_dyu[NV * VEC];
#pragma unroll
  for (int i = 0; i < NV * VEC; ++i)
    sum_dy[i] = sum_dyu[i] = 0.0f;
  Pack<P, VEC> g[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    g[i] = cols.template parameter<P>(gamma + cols.first, i, gamma != nullptr, 1.0f);
  Pack<T, VEC> next_x[NV], next_dy[NV];
  float next_mean = 0.0f, next_var = 0.0f;
  auto fetch = [&](int64_t row) {
    const T *xr = x + row * size + cols.first, *dr = dy + row * size + cols.first;
#pragma unroll
    for (int i = 0; i < NV; ++i) { // (beyond the row a dy of 0 adds nothing to any sum)
      next_x[i] = cols.template load<T, true>(xr, i);
      next_dy[i] = cols.template load<T, true>(dr, i);
    }
    next_mean = mean[row], next_var = var[row];
  };
  if (first < rows)
    fetch(first);
  int turn = 0;
  for (int64_t row = first; row < rows; row += stride) {
    Pack<T, VEC> xv[NV], dv[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i)
      xv[i] = next_x[i], dv[i] = next_dy[i];
    const float mu = next_mean, r = rsqrtf(next_var + eps);
    if (row + stride < rows)
      fetch(row + stride);
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float u = (xv[i].f(j) - mu) * r, d = dv[i].f(j), gd = d * g[i].f(j);
        s[0] += gd;
        s[1] = fmaf(gd, u, s[1]);
        if (kParams) {
          sum_dy[i * VEC + j] += d;
          sum_dyu[i * VEC + j] = fmaf(d, u, sum_dyu[i * VEC + j]);
        }
      }
    if (!dx)
      continue;
    row_sums<2>(s, row_warps, slots, turn);
    if constexpr (kCluster)
      cluster_sums<2>(s, shared_sums[turn], cluster); // (turn alternates: the other slot's readers have passed its barrier)
    // r (gd - m1 - u m2) as r gd + (a x + b)
    const float m1 = s[0] * inv_size, a = -r * r * (s[1] * inv_size), b = fmaf(-mu, a, -r * m1);
    T *out = dx + row * size + cols.first;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!cols.some(i))
        continue;
      float o[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        o[j] = fmaf(dv[i].f(j) * g[i].f(j), r, fmaf(xv[i].f(j), a, b));
      if (accum) {
        const Pack<T, VEC> old = cols.template load<T, false>(out, i);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          o[j] += old.f(j);
      }
      cols.store(out, i, o, keep);
    }
  }
  if constexpr (kParams) {
    float *mine = partial + block * 2 * size, *own = row_warps > 1 ? mine : combine + (size_t)warp * 2 * size;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (cols.some(i))
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (cols.has(i, j)) {
            own[cols.at(i) + j] = sum_dy[i * VEC + j];
            own[size + cols.at(i) + j] = sum_dyu[i * VEC + j];
          }
    if (row_warps == 1) {
      __syncthreads();
      for (int c = threadIdx.x; c < 2 * size; c += blockDim.x) {
        float s = 0.0f;
        for (int w = 0; w < warps; ++w)
          s += combine[(size_t)w * 2 * size + c];
        mine[c] = s;
      }
    }
  }
  if constexpr (kCluster) // no block leaves while another may still read its sums
    cluster_barrier();
}

// The same sums for rows too long for the kernel above: a thread a column, a slab of rows a block, partial sums
// [slabs][2][size].
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_columns_kernel(const T *__restrict__ x, const T *__restrict__ dy,
                                                                 const float *__restrict__ mean,
                                                                 const float *__restrict__ var,
                                                                 float *__restrict__ partial, int64_t rows, int64_t size,
                                                                 int64_t slab, float eps) {
  pdl_wait();
  pdl_trigger();
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= size)
    return;
  const int64_t r0 = blockIdx.y * slab, r1 = r0 + slab < rows ? r0 + slab : rows;
  float a = 0.0f, b = 0.0f;
#pragma unroll 4
  for (int64_t row = r0; row < r1; ++row) {
    const float d = to_f32(dy[row * size + c]);
    a += d;
    b = fmaf(d, (to_f32(x[row * size + c]) - mean[row]) * (rsqrtf(var[row] + eps)), b);
  }
  partial[(int64_t)blockIdx.y * 2 * size + c] = a;
  partial[(int64_t)blockIdx.y * 2 * size + size + c] = b;
}

// dbeta (+)= sum over the parts of [part][0][c], dgamma of [part][1][c], in a fixed order: `share` of a block's 32 warps take the
// parts of 32 columns in turn.
template <typename P>
__global__ void __launch_bounds__(1024) layer_norm_param_kernel(const float *__restrict__ partial, int parts, int share,
                                                                int64_t size, P *dbeta, P *dgamma, bool accum_beta,
                                                                bool accum_gamma) {
  __shared__ float sums[32][33];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = warp % share;
  P *out = blockIdx.y == 0 ? dbeta : dgamma;
  if (!out)
    return;
  const bool accum = blockIdx.y == 0 ? accum_beta : accum_gamma;
  const int64_t c = ((int64_t)blockIdx.x * (32 / share) + warp / share) * 32 + lane;
  float s = 0.0f;
  if (c < size) {
    const float *p = partial + (int64_t)blockIdx.y * size + c;
#pragma unroll 8
    for (int k = mine; k < parts; k += share)
      s += p[(int64_t)k * 2 * size];
  }
  sums[warp][lane] = s;
  __syncthreads();
  if (mine == 0 && c < size) {
    for (int w = 1; w < share; ++w)
      s += sums[warp + w][lane];
    if (accum)
      s += to_f32(out[c]);
    out[c] = from_f32<P>(s);
  }
}

// Threads of a row, accesses of a thread, and blocks of a cluster that share a row. Rows of up to four accesses a lane are a
// warp's (no barrier); longer ones a block's, with `want` accesses a thread where the rows are enough to fill the SMs and one
// where they are few, and of up to eight blocks where one does not hold them in registers, or where the rows leave SMs idle.
struct RowShape {
  int row_warps, nv, cluster;
  int64_t slice; // columns of a cluster's block
  bool fits;
};
RowShape row_shape(int64_t size, int vec, bool shift, int64_t rows, int max_nv, int want) {
  const int64_t packs = (size + (shift ? vec - 1 : 0) + vec - 1) / vec;
  if (packs <= 32)
    return {1, 1, 1, 0, true};
  const bool few = rows < 2 * sm_count();
  if (packs <= 32 * std::min(4, max_nv) && !few)
    return {1, packs <= 64 ? 2 : 4, 1, 0, true};
  // (in a cluster 256 threads a block: several rows an SM hide the latency of their barriers)
  const int64_t most = packs > 512 * max_nv ? 256 * max_nv : 512 * max_nv;
  int cluster = 1;
  while (cluster < 8 && ((packs + cluster - 1) / cluster > most || (rows * cluster < sm_count() && packs >= 1024 * cluster)))
    cluster *= 2;
  const int64_t each = (packs + cluster - 1) / cluster;
  int threads = 128;
  while (threads < 512 && (int64_t)threads * (few ? 1 : want) < each)
    threads *= 2;
  int nv = 1;
  while (nv < max_nv && (int64_t)threads * nv < each)
    nv *= 2;
  return {threads / 32, nv, cluster, each * vec, (int64_t)threads * nv >= each};
}

template <int... N, typename F> int with_count(int n, std::integer_sequence<int, N...>, F f) {
  int rc = NB200_EVALUE;
  ((n == N ? (rc = f(std::integral_constant<int, N>{}), 0) : 0), ...);
  return rc;
}
using Counts = std::integer_sequence<int, 1, 2, 4, 8, 16>;

int check_sizes(int64_t rows, int64_t size, int64_t per_row_blocks) {
  NB_CHECK(size > 0, NB200_EVALUE, "an empty row has no mean");
  NB_CHECK(size < (1ll << 31), NB200_EVALUE, "a row has 2^31 values or more");
  NB_CHECK(rows >= 0 && rows * per_row_blocks < (1ll << 31), NB200_EVALUE, "too many rows");
  return NB200_OK;
}

// How rows are accessed: 16 bytes at a time, from boundaries in front of the rows where their size is no multiple of that, or
// (tensors that begin off a boundary) value by value.
template <typename T, typename F> int with_access(int64_t size, bool aligned_rows, bool aligned_params, F f) {
  if (!aligned_rows || (size % kPackOf<T> == 0 && !aligned_params))
    return f(std::integral_constant<int, 1>{}, std::false_type{});
  return size % kPackOf<T> == 0 ? f(std::integral_constant<int, kPackOf<T>>{}, std::false_type{})
                                : f(std::integral_constant<int, kPackOf<T>>{}, std::true_type{});
}

template <typename T, typename P>
int forward(const T *x, const P *beta, const P *gamma, T *y, float *mean, float *var, int64_t rows, int64_t size, float eps,
            cudaStream_t st) {
  const bool keep = (size_t)rows * size * sizeof(T) <= kKeepBytes;
  return with_access<T>(size, aligned16(x) && aligned16(y), aligned16(gamma) && aligned16(beta), [&](auto vec, auto shift) -> int {
    constexpr int kVec = decltype(vec)::value, kMaxNv = kVec == 1 ? 16 : kVec == 4 ? 8 : 4;
    constexpr bool kShift = decltype(shift)::value;
    const RowShape s = row_shape(size, kVec, kShift, rows, kMaxNv, kVec == 1 ? 8 : 4);
    if (!s.fits) {
      NB_CUDA(launch_dependent(layer_norm_long_kernel<T, P, false>, dim3((unsigned)(rows * kLongBlocks)), dim3(kLongThreads),
                               0, st, x, (const T *)nullptr, beta, gamma, y, mean, var, size, eps, false));
      return NB200_OK;
    }
    const int per_block = s.row_warps == 1 ? 4 : 1;
    return with_count(s.nv, Counts{}, [&](auto nv) -> int {
      constexpr int kNv = decltype(nv)::value;
      auto launch = [&](auto count, auto clustered) -> int {
        constexpr int kRows = decltype(count)::value;
        const int64_t blocks = (rows + per_block * kRows - 1) / (per_block * kRows);
        auto kernel = layer_norm_kernel<T, P, kVec, kNv, kRows, kShift, decltype(clustered)::value>;
        const int threads = 32 * s.row_warps * per_block;
        if (decltype(clustered)::value)
          NB_CUDA(launch_clusters(kernel, (unsigned)(blocks * s.cluster), s.cluster, threads, 0, st, x, beta, gamma, y, mean, var,
                                  rows, (int)size, 1.0f / (float)size, eps, s.row_warps, s.cluster, (int)s.slice, keep));
        else
          NB_CUDA(launch_dependent(kernel, dim3((unsigned)blocks), dim3(threads), 0, st, x, beta, gamma, y, mean, var, rows,
                                   (int)size, 1.0f / (float)size, eps, s.row_warps, 1, 0, keep));
        return NB200_OK;
      };
      if constexpr (kNv <= kMaxNv) {
        if (s.cluster > 1)
          return launch(std::integral_constant<int, 1>{}, std::true_type{});
        if constexpr (!kShift && kVec * kNv <= 16)
          if (rows / per_block >= 64 * sm_count()) // two rows at once where that leaves enough blocks
            return launch(std::integral_constant<int, 2>{}, std::false_type{});
        return launch(std::integral_constant<int, 1>{}, std::false_type{});
      }
      return NB200_EVALUE;
    });
  });
}

template <typename T, typename P>
int backward(const T *x, const T *dy, const P *gamma, const float *mean, const float *var, T *dx, P *dbeta, P *dgamma,
             int64_t rows, int64_t size, float eps, bool accum_dx, bool accum_beta, bool accum_gamma, cudaStream_t st) {
  const bool params = dbeta || dgamma, keep = (size_t)rows * size * sizeof(T) <= kKeepBytes;
  AsyncScratch scratch(st);
  int parts = 0;
  auto run = [&](auto vec, auto shift) -> int {
    constexpr int kVec = decltype(vec)::value, kMaxNv = kVec == 1 ? 16 : kVec == 4 ? 4 : 2;
    constexpr bool kShift = decltype(shift)::value;
    RowShape s = row_shape(size, kVec, kShift, rows, kMaxNv, kVec == 1 ? 8 : 2);
    const bool walk = s.fits && s.cluster == 1; // one kernel for dx and the sums over the rows
    if (!walk) // (without those sums a thread has room for twice as much of a row)
      s = row_shape(size, kVec, kShift, rows, std::min(16, 2 * kMaxNv), kVec == 1 ? 8 : 4);
    if (!walk && params) {
      const int64_t columns = (size + 255) / 256;
      const int64_t slabs = std::max<int64_t>(1, std::min<int64_t>((rows + 7) / 8, 8 * sm_count() / columns));
      const int64_t slab = (rows + slabs - 1) / slabs;
      parts = (int)((rows + slab - 1) / slab);
      NB_TRY(scratch.alloc((size_t)parts * 2 * size * 4));
      NB_CUDA(launch_dependent(layer_norm_columns_kernel<T>, dim3((unsigned)columns, (unsigned)parts), dim3(256), 0, st, x, dy,
                               mean, var, static_cast<float *>(scratch.p), rows, size, slab, eps));
    }
    if (!walk && !dx)
      return NB200_OK;
    if (!s.fits) { // (after the sums: it may overwrite x or dy)
      NB_CUDA(launch_dependent(layer_norm_long_kernel<T, P, true>, dim3((unsigned)(rows * kLongBlocks)), dim3(kLongThreads), 0, st,
                               x, dy, (const P *)nullptr, gamma, dx, const_cast<float *>(mean), const_cast<float *>(var), size,
                               eps, accum_dx));
      return NB200_OK;
    }
    const int per_block = s.row_warps == 1 ? 8 : 1, threads = 32 * s.row_warps * per_block;
    // As many blocks as are resident, and then no more than their rounds need: each leaves partial sums. With kShift a multiple
    // of VEC, where any has a second row.
    const int64_t groups = (rows + per_block - 1) / per_block, most = (int64_t)sm_count() * std::max(1, 512 / threads);
    const int64_t rounds = walk ? (groups + most - 1) / most : 1;
    int64_t blocks = (groups + rounds - 1) / rounds;
    if (kShift && rounds > 1)
      blocks = (blocks + kVec - 1) / kVec * kVec;
    if (walk && params) {
      parts = (int)blocks;
      NB_TRY(scratch.alloc((size_t)parts * 2 * size * 4));
    }
    return with_count(s.nv, Counts{}, [&](auto nv) -> int {
      constexpr int kNv = decltype(nv)::value;
      const size_t smem = walk && params && s.row_warps == 1 ? (size_t)per_block * 2 * size * 4 : 0;
      static_assert(8 * 2 * 32 * std::min(4, kMaxNv) * kVec * 4 <= 48 * 1024, "a warp's rows need no opt-in");
      auto launch = [&](auto kernel, auto clustered) -> int {
        if (decltype(clustered)::value)
          NB_CUDA(launch_clusters(kernel, (unsigned)(blocks * s.cluster), s.cluster, threads, smem, st, x, dy, gamma, mean, var, dx,
                                  static_cast<float *>(nullptr), rows, (int)size, 1.0f / (float)size, eps, s.row_warps, s.cluster,
                                  (int)s.slice, accum_dx, keep));
        else
          NB_CUDA(launch_dependent(kernel, dim3((unsigned)blocks), dim3(threads), smem, st, x, dy, gamma, mean, var, dx,
                                   static_cast<float *>(scratch.p), rows, (int)size, 1.0f / (float)size, eps, s.row_warps, 1, 0,
                                   accum_dx, keep));
        return NB200_OK;
      };
      if constexpr (kNv <= kMaxNv)
        if (walk && params)
          return launch(layer_norm_backward_kernel<T, P, kVec, kNv, true, kShift, false>, std::false_type{});
      if constexpr (kNv <= 2 * kMaxNv && kNv <= 16)
        return s.cluster > 1 ? launch(layer_norm_backward_kernel<T, P, kVec, kNv, false, kShift, true>, std::true_type{})
                             : launch(layer_norm_backward_kernel<T, P, kVec, kNv, false, kShift, false>, std::false_type{});
      return NB200_EVALUE;
    });
  };
  if (rows > 0)
    NB_TRY(with_access<T>(size, aligned16(x) && aligned16(dy) && aligned16(dx), aligned16(gamma), run));
  if (params) {
    int share = 1;
    while (share < 32 && share < parts)
      share *= 2;
    const int64_t columns = 32 * (32 / share);
    NB_CUDA(launch_dependent(layer_norm_param_kernel<P>, dim3((unsigned)((size + columns - 1) / columns), 2), dim3(1024), 0, st,
                             static_cast<const float *>(scratch.p), parts, share, size, dbeta, dgamma, accum_beta, accum_gamma));
  }
  return NB200_OK;
}

// f(T{}, P{}) for a type and a parameter type that is the same or fp32
template <typename F> int with_types(int type, int param_type, F f) {
  NB_CHECK(param_type == type || param_type == NB200_F32, NB200_EVALUE, "beta and gamma have x's type or float32");
  return with_type(type, [&](auto t) -> int {
    using T = decltype(t);
    return param_type == type ? f(T{}, T{}) : f(T{}, float{});
  });
}

} // namespace
} // namespace nb200

using namespace nb200;

extern "C" int nb200_layer_normalization(const void *x, const void *beta, const void *gamma, void *y, float *mean,
                                         float *variance, int64_t rows, int64_t size, float eps, int type, int param_type,
                                         void *stream) {
  NB_TRY(check_sizes(rows, size, kLongBlocks));
  if (rows == 0)
    return NB200_OK;
  NB_CHECK(x && y, NB200_EVALUE, "null data pointer");
  return with_types(type, param_type, [&](auto t, auto p) {
    using T = decltype(t);
    using P = decltype(p);
    return forward<T, P>(static_cast<const T *>(x), static_cast<const P *>(beta), static_cast<const P *>(gamma),
                         static_cast<T *>(y), mean, variance, rows, size, eps, as_stream(stream));
  });
}

extern "C" int nb200_layer_normalization_backward(const void *x, const void *dy, const void *gamma, const float *mean,
                                                  const float *variance, void *dx, void *dbeta, void *dgamma, int64_t rows,
                                                  int64_t size, float eps, int type, int param_type, int accum_dx,
                                                  int accum_dbeta, int accum_dgamma, void *stream) {
  NB_TRY(check_sizes(rows, size, kLongBlocks));
  NB_CHECK(rows == 0 || (x && dy && mean && variance), NB200_EVALUE, "null data pointer");
  if (!dx && !dbeta && !dgamma)
    return NB200_OK;
  return with_types(type, param_type, [&](auto t, auto p) {
    using T = decltype(t);
    using P = decltype(p);
    return backward<T, P>(static_cast<const T *>(x), static_cast<const T *>(dy), static_cast<const P *>(gamma), mean,
                          variance, static_cast<T *>(dx), static_cast<P *>(dbeta), static_cast<P *>(dgamma), rows, size, eps,
                          accum_dx != 0, accum_dbeta != 0, accum_dgamma != 0, as_stream(stream));
  });
}
