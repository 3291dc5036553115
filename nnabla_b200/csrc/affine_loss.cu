// Softmax cross entropy of an affine layer's classes, l = x W + b [rows, classes], without keeping l:
//
//   loss = log sum_v exp(l_v) - l_label
//   G_v = (exp(l_v) / sum_u exp(l_u) - [v = label]) dloss;  dx = G W^T, dW = x^T G, db = sum over rows of G
//
// Forward: a product whose epilogue leaves, of each row and tile of classes, the maximum and the sum of the exponentials, and
// the label's logit; a second kernel joins them. Backward, for a piece of the classes after the other: the product again,
// with G as its result, then the two products with G. The label of a row that does not count is negative: its loss and its
// row of G are 0. A label >= classes makes its row's loss, and every gradient that it enters, NaN.
#include <algorithm>

#include "pdl.cuh"
#include "softmax_sums.cuh"

namespace nb200 {
namespace {

// What becomes of a tile of the logits. kSums: partial[row][tile of classes] and the label's logit. kGrad: G.
struct Rows {
  const void *label; // label_bytes each
  int label_bytes;
  const float2 *stat; // kGrad: of the forward pass
  const float *dloss;
  float2 *partial; // kSums: [rows][tiles]
  float *target;
  int tiles;
  int64_t classes;
  __device__ __forceinline__ int64_t label_of(int64_t row) const {
    return label_bytes == 8 ? static_cast<const int64_t *>(label)[row] : (int64_t) static_cast<const int32_t *>(label)[row];
  }
};

// ---- products on the CUDA cores ------------------------------------------------------------------------------------------
// D[m, n] = sum_k A(m, k) B(k, n) with any strides, in fp32: 64 x 64 tiles, 16 of K at a time, 4 x 4 results a thread.
template <typename T> struct Strided {
  const T *p;
  int64_t row, col;
};
enum class Out { kSums, kGrad, kStore };

template <typename TA, typename TB, typename TO, Out kOut>
__global__ void __launch_bounds__(256) simt_product_kernel(Strided<TA> a, Strided<TB> b, int64_t M, int64_t N, int64_t K,
                                                           const TO *__restrict__ bias, Rows rows, int64_t class0, TO *out,
                                                           int64_t ldo, bool accum) {
  __shared__ float as[16][65], bs[16][65];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < K; k0 += 16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // neighbouring threads along the axis that lies in neighbouring memory
      const int e = tid + i * 256;
      const int am = a.col == 1 ? e >> 4 : e & 63, ak = a.col == 1 ? e & 15 : e >> 6;
      as[ak][am] = m0 + am < M && k0 + ak < K ? to_f32(a.p[(m0 + am) * a.row + (k0 + ak) * a.col]) : 0.0f;
      const int bn = b.col == 1 ? e & 63 : e >> 4, bk = b.col == 1 ? e >> 6 : e & 15;
      bs[bk][bn] = n0 + bn < N && k0 + bk < K ? to_f32(b.p[(k0 + bk) * b.row + (n0 + bn) * b.col]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      float u[4], v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u[i] = as[k][ty * 4 + i];
        v[i] = bs[k][tx * 4 + i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = fmaf(u[i], v[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty * 4 + i;
    if constexpr (kOut == Out::kStore) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t n = n0 + tx * 4 + j;
        if (m < M && n < N) {
          TO *to = out + m * ldo + n;
          *to = from_f32<TO>(accum ? to_f32(*to) + acc[i][j] : acc[i][j]);
        }
      }
    } else {
      const int64_t label = m < M ? rows.label_of(m) : -1;
      MaxSum t{-INFINITY, 0.0f};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t n = n0 + tx * 4 + j;
        if (m >= M || n >= N)
          continue;
        const float l = bias ? acc[i][j] + to_f32(bias[class0 + n]) : acc[i][j];
        if constexpr (kOut == Out::kSums) {
          t = join(t, MaxSum{l, l == -INFINITY ? 0.0f : 1.0f}, kLog2e);
          if (l != l)
            t.s = l;
          if (class0 + n == label)
            rows.target[m] = l;
        } else {
          const float2 st = rows.stat[m];
          float g = ex2(fmaf(l - st.x, kLog2e, -st.y * kLog2e));
          g -= class0 + n == label ? 1.0f : 0.0f;
          reinterpret_cast<float *>(out)[m * ldo + n] = label < 0 ? 0.0f : label >= rows.classes ? NAN : g * rows.dloss[m];
        }
      }
      if constexpr (kOut == Out::kSums) {
#pragma unroll
        for (int d = 8; d; d >>= 1)
          t = join(t, MaxSum{__shfl_xor_sync(0xffffffffu, t.m, d), __shfl_xor_sync(0xffffffffu, t.s, d)}, kLog2e);
        if (tx == 0 && m < M)
          rows.partial[m * rows.tiles + blockIdx.x] = make_float2(t.m, t.s);
      }
    }
  }
}

// The rows' loss and statistics from the tiles' maxima and sums: a warp a row.
__global__ void __launch_bounds__(256) loss_rows_kernel(Rows rows, int64_t count, float *__restrict__ loss,
                                                        float2 *__restrict__ stat) {
  pdl_wait();
  pdl_trigger();
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= count)
    return;
  MaxSum t{-INFINITY, 0.0f};
  for (int i = lane; i < rows.tiles; i += 32) {
    const float2 p = rows.partial[row * rows.tiles + i];
    t = join(t, MaxSum{p.x, p.y}, kLog2e);
  }
  t = warp_join(t, kLog2e);
  if (lane == 0) {
    const int64_t label = rows.label_of(row);
    const float log_sum = log2f(t.s) * kLn2;
    stat[row] = make_float2(t.m, log_sum);
    loss[row] = label < 0 ? 0.0f : label >= rows.classes ? NAN : (t.m - rows.target[row]) + log_sum;
  }
}

// db (+)= the column sums of G, a block 32 columns.
template <typename G, typename TO>
__global__ void __launch_bounds__(512) column_sums_kernel(const G *__restrict__ g, int64_t rows, int64_t columns, int64_t ld,
                                                          TO *db, bool accum) {
  __shared__ float sums[16][33];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (c < columns)
    for (int64_t r = warp; r < rows; r += 16)
      s += to_f32(g[r * ld + c]);
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < columns) {
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w)
      s += sums[w][lane];
    db[c] = from_f32<TO>(accum ? s + to_f32(db[c]) : s);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) round_kernel(const float *__restrict__ from, T *to, int64_t n, bool accum) {
  pdl_wait();
  pdl_trigger();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    to[i] = from_f32<T>(accum ? from[i] + to_f32(to[i]) : from[i]);
}

template <typename T>
int forward(const T *x, const T *w, const T *bias, const void *label, int label_bytes, float *loss, float2 *stat,
            int64_t rows, int64_t size, int64_t classes, cudaStream_t st) {
  const int64_t tiles = (classes + 63) / 64;
  AsyncScratch scratch(st);
  NB_TRY(scratch.alloc((size_t)rows * tiles * 8 + (size_t)rows * 4));
  Rows r{};
  r.label = label, r.label_bytes = label_bytes, r.classes = classes, r.tiles = (int)tiles;
  r.partial = static_cast<float2 *>(scratch.p);
  r.target = reinterpret_cast<float *>(r.partial + rows * tiles);
  NB_CUDA(launch_dependent(simt_product_kernel<T, T, T, Out::kSums>, dim3((unsigned)tiles, (unsigned)((rows + 63) / 64)),
                           dim3(256), 0, st, Strided<T>{x, size, 1}, Strided<T>{w, classes, 1}, rows, classes, size, bias, r,
                           (int64_t)0, (T *)nullptr, (int64_t)0, false));
  NB_CUDA(launch_dependent(loss_rows_kernel, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, r, rows, loss, stat));
  return NB200_OK;
}

template <typename T>
int backward(const T *x, const T *w, const T *bias, const void *label, int label_bytes, const float2 *stat,
             const float *dloss, T *dx, T *dw, T *db, int64_t rows, int64_t size, int64_t classes, const bool accum[3],
             cudaStream_t st) {
  const int64_t piece = std::max<int64_t>(64, std::min<int64_t>((classes + 63) / 64 * 64, (16 << 20) / rows / 64 * 64));
  const bool pieces = piece < classes;
  AsyncScratch scratch(st);
  NB_TRY(scratch.alloc((size_t)rows * piece * 4 + (pieces && dx ? (size_t)rows * size * 4 : 0)));
  float *g = static_cast<float *>(scratch.p), *dx32 = g + rows * piece;
  Rows r{};
  r.label = label, r.label_bytes = label_bytes, r.classes = classes, r.stat = stat, r.dloss = dloss;
  for (int64_t c0 = 0; c0 < classes; c0 += piece) {
    const int64_t n = std::min(piece, classes - c0);
    NB_CUDA(launch_dependent(simt_product_kernel<T, T, T, Out::kGrad>,
                             dim3((unsigned)((n + 63) / 64), (unsigned)((rows + 63) / 64)), dim3(256), 0, st,
                             Strided<T>{x, size, 1}, Strided<T>{w + c0, classes, 1}, rows, n, size, bias, r, c0,
                             reinterpret_cast<T *>(g), piece, false));
    if (dx) {
      const dim3 grid((unsigned)((size + 63) / 64), (unsigned)((rows + 63) / 64));
      if (pieces)
        NB_CUDA(launch_dependent(simt_product_kernel<float, T, float, Out::kStore>, grid, dim3(256), 0, st,
                                 Strided<float>{g, piece, 1}, Strided<T>{w + c0, 1, classes}, rows, size, n,
                                 (const float *)nullptr, r, c0, dx32, size, c0 > 0));
      else
        NB_CUDA(launch_dependent(simt_product_kernel<float, T, T, Out::kStore>, grid, dim3(256), 0, st,
                                 Strided<float>{g, piece, 1}, Strided<T>{w + c0, 1, classes}, rows, size, n,
                                 (const T *)nullptr, r, c0, dx, size, accum[0]));
    }
    if (dw)
      NB_CUDA(launch_dependent(simt_product_kernel<T, float, T, Out::kStore>,
                               dim3((unsigned)((n + 63) / 64), (unsigned)((size + 63) / 64)), dim3(256), 0, st,
                               Strided<T>{x, 1, size}, Strided<float>{g, piece, 1}, size, n, rows, (const T *)nullptr, r, c0,
                               dw + c0, classes, accum[1]));
    if (db)
      NB_CUDA(launch_dependent(column_sums_kernel<float, T>, dim3((unsigned)((n + 31) / 32)), dim3(512), 0, st,
                               (const float *)g, rows, n, piece, db + c0, accum[2]));
  }
  if (dx && pieces)
    NB_CUDA(launch_dependent(round_kernel<T>, dim3((unsigned)std::min<int64_t>((rows * size + 255) / 256, 8 * sm_count())),
                             dim3(256), 0, st, (const float *)dx32, dx, rows * size, accum[0]));
  return NB200_OK;
}

int check(int64_t rows, int64_t size, int64_t classes, int label_bytes) {
  NB_CHECK(rows >= 0 && rows < (1ll << 22), NB200_EVALUE, "%lld rows outside [0, 2^22)", (long long)rows);
  NB_CHECK(size > 0 && size < (1ll << 24), NB200_EVALUE, "%lld inputs outside [1, 2^24)", (long long)size);
  NB_CHECK(classes > 0 && classes < (1ll << 24), NB200_EVALUE, "%lld classes outside [1, 2^24)", (long long)classes);
  NB_CHECK(label_bytes == 4 || label_bytes == 8, NB200_EVALUE, "labels are 4 or 8 byte integers, not %d", label_bytes);
  return NB200_OK;
}

} // namespace
} // namespace nb200

using namespace nb200;

extern "C" int nb200_affine_softmax_cross_entropy(const void *x, const void *w, const void *bias, const void *label,
                                                  float *loss, float *stat, int64_t rows, int64_t size, int64_t classes,
                                                  int type, int label_bytes, void *stream) {
  NB_TRY(check(rows, size, classes, label_bytes));
  if (rows == 0)
    return NB200_OK;
  NB_CHECK(x && w && label && loss && stat, NB200_EVALUE, "null data pointer");
  NB_CHECK((reinterpret_cast<uintptr_t>(stat) & 7) == 0, NB200_EVALUE, "stat holds pairs: 8-byte aligned");
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    return forward<T>(static_cast<const T *>(x), static_cast<const T *>(w), static_cast<const T *>(bias), label, label_bytes,
                      loss, reinterpret_cast<float2 *>(stat), rows, size, classes, as_stream(stream));
  });
}

extern "C" int nb200_affine_softmax_cross_entropy_backward(const void *x, const void *w, const void *bias, const void *label,
                                                           const float *stat, const float *dloss, void *dx, void *dw,
                                                           void *db, int64_t rows, int64_t size, int64_t classes, int type,
                                                           int label_bytes, int accum_dx, int accum_dw, int accum_db,
                                                           void *stream) {
  NB_TRY(check(rows, size, classes, label_bytes));
  if (rows == 0) { // sums over no rows
    if (dw && !accum_dw)
      NB_CUDA(cudaMemsetAsync(dw, 0, (size_t)size * classes * type_bytes(type), as_stream(stream)));
    if (db && !accum_db)
      NB_CUDA(cudaMemsetAsync(db, 0, (size_t)classes * type_bytes(type), as_stream(stream)));
    return NB200_OK;
  }
  if (!dx && !dw && !db)
    return NB200_OK;
  NB_CHECK(x && w && label && stat && dloss, NB200_EVALUE, "null data pointer");
  NB_CHECK((reinterpret_cast<uintptr_t>(stat) & 7) == 0, NB200_EVALUE, "stat holds pairs: 8-byte aligned");
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    const bool accum[3] = {accum_dx != 0, accum_dw != 0, accum_db != 0};
    return backward<T>(static_cast<const T *>(x), static_cast<const T *>(w), static_cast<const T *>(bias), label, label_bytes,
                       reinterpret_cast<const float2 *>(stat), dloss, static_cast<T *>(dx), static_cast<T *>(dw),
                       static_cast<T *>(db), rows, size, classes, accum, as_stream(stream));
  });
}
