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

#include "few_rows.cuh"
#include "loss_gemm.cuh"
#include "prepare.cuh"

namespace nb200 {
namespace {

// The rows' loss and statistics from the tiles' maxima and sums: a warp a row.
__global__ void __launch_bounds__(256) loss_rows_kernel(LossRows rows, int64_t count, float *__restrict__ loss,
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

// db (+)= the column sums of G, [planes][rows][ld], a block 32 columns; scale[2] (scale NULL: 1) undoes G's scaling.
template <typename G, typename TO>
__global__ void __launch_bounds__(512) column_sums_kernel(const G *__restrict__ g, int planes, int64_t rows, int64_t columns,
                                                          int64_t ld, const float *scale, TO *db, bool accum) {
  __shared__ float sums[16][33];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (c < columns)
#pragma unroll 8
    for (int64_t r = warp; r < planes * rows; r += 16)
      s += to_f32(g[r * ld + c]);
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < columns) {
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w)
      s += sums[w][lane];
    if (scale)
      s *= scale[2];
    db[c] = from_f32<TO>(accum ? s + to_f32(db[c]) : s);
  }
}

// to (+)= the sum of `parts` tensors of n values, in order.
template <typename T>
__global__ void __launch_bounds__(256) round_kernel(const float *__restrict__ from, int parts, T *to, int64_t n, bool accum) {
  pdl_wait();
  pdl_trigger();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float s = 0.0f;
    for (int p = 0; p < parts; ++p)
      s += from[p * n + i];
    to[i] = from_f32<T>(accum ? s + to_f32(to[i]) : s);
  }
}

// [rows][cols] -> [rows][pitch] of 16-bit values, for rows that a TMA copy cannot read where they lie; eight values a thread.
__global__ void __launch_bounds__(256) repitch_kernel(const uint16_t *__restrict__ from, uint16_t *__restrict__ to,
                                                      int64_t rows, int64_t cols, int64_t pitch) {
  pdl_wait();
  pdl_trigger();
  const int64_t packs = pitch / 8;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * packs; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / packs, c = (i - r * packs) * 8;
    Pack<uint16_t, 8> v;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v.v[j] = c + j < cols ? from[r * cols + c + j] : (uint16_t)0;
    *reinterpret_cast<Pack<uint16_t, 8> *>(to + r * pitch + c) = v;
  }
}

// What G is kept relative to: scale = {the largest |dloss| of a row that counts, 2^e, their quotient}. With the largest taken
// out, the gradient of a mean, the same in every row, is no rounded factor of G: at the label G is -1 + p. e is 14 for an fp16 G,
// which so has eleven bits down to 2^-28 of the largest gradient, and 0 for the others.
__global__ void __launch_bounds__(1024) gradient_scale_kernel(LossRows rows, int64_t count, float times, float *scale) {
  __shared__ float tops[32];
  pdl_wait();
  pdl_trigger();
  float top = 0.0f;
  for (int64_t r = threadIdx.x; r < count; r += 1024)
    if (rows.label_of(r) >= 0)
      top = fmaxf(top, fabsf(rows.dloss[r]));
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0)
    tops[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x < 32) {
    top = warp_max(tops[threadIdx.x]);
    if (threadIdx.x == 0) {
      // (none, or one that is not finite: G as it is)
      const bool plain = !(top >= 1.17549435e-38f && top < INFINITY);
      scale[0] = plain ? 1.0f : top;
      scale[1] = times;
      scale[2] = (plain ? 1.0f : top) / times;
    }
  }
}

int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// A matrix as an operand of the tensor-core products: as it lies, or (rows that a TMA copy cannot read, fp32) laid out anew
// in `scratch`, of operand_bytes().
template <typename T> size_t operand_bytes(const T *p, int64_t rows, int64_t cols) {
  if (std::is_same<T, float>::value)
    return (size_t)3 * rows * up(cols, 64) * 2;
  return cols % 8 == 0 && aligned16(p) ? 0 : (size_t)rows * up(cols, 8) * 2;
}
template <typename T> int make_operand(const T *p, int64_t rows, int64_t cols, void *scratch, Operand &o, cudaStream_t st) {
  o = {scratch, rows, cols, up(cols, std::is_same<T, float>::value ? 64 : 8), 1};
  if constexpr (std::is_same<T, float>::value) {
    o.planes = 3;
    return split_rows_bf16(SplitRows{p, nullptr, scratch, rows, (int)cols, 3}, SplitRows{}, o.pitch, st);
  } else if (operand_bytes(p, rows, cols) == 0) {
    o.p = p;
  } else {
    const int64_t blocks = (rows * (o.pitch / 8) + 255) / 256;
    NB_CUDA(launch_dependent(repitch_kernel, dim3((unsigned)std::min<int64_t>(blocks, 64 * sm_count())), dim3(256), 0, st,
                             reinterpret_cast<const uint16_t *>(p), static_cast<uint16_t *>(scratch), rows, cols, o.pitch));
  }
  return NB200_OK;
}
Operand columns(Operand o, int64_t c0, int64_t n) {
  o.p = static_cast<const char *>(o.p) + 2 * c0;
  o.cols = n;
  return o;
}

// Time of a launch's tiles, in MMA cycles of an SM: rounds of 256 x 256 tiles on pairs of SMs, 512 cycles a K block, or of
// 128 x 64 ones, 204 (51 an instruction, for its operands' reads; 32 by its products).
struct TileCount {
  int64_t M, N, kblocks;
};
bool pays_pairs(std::initializer_list<TileCount> products) {
  int64_t pair_tiles = 0, single_tiles = 0, blocks = 1;
  for (const TileCount &p : products) {
    pair_tiles += ((p.M + 255) / 256) * ((p.N + 255) / 256);
    single_tiles += ((p.M + 127) / 128) * ((p.N + 63) / 64);
    blocks = std::max(blocks, p.kblocks);
  }
  auto rounds = [](int64_t tiles, int64_t units) { return (tiles + units - 1) / units; };
  return rounds(pair_tiles, sm_count() / 2) * 512 <= rounds(single_tiles, sm_count()) * 204;
}

// Scratch for a call, in parts that begin at 256-byte boundaries.
struct Parts {
  size_t bytes = 0;
  size_t take(size_t n) {
    const size_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  }
};

template <typename T>
int forward_tensor(const T *x, const T *w, const T *bias, LossRows r, float *loss, float2 *stat, int64_t rows, int64_t size,
                   int64_t classes, cudaStream_t st) {
  const int kblocks = (int)((size + 63) / 64);
  const bool pair = pays_pairs({{rows, classes, kblocks}});
  r.tiles = (int)(2 * ((classes + (pair ? 255 : 63)) / (pair ? 256 : 64)));
  Parts parts;
  const size_t at_x = parts.take(operand_bytes(x, rows, size)), at_w = parts.take(operand_bytes(w, size, classes));
  const size_t at_partial = parts.take((size_t)rows * r.tiles * 8), at_target = parts.take((size_t)rows * 4);
  AsyncScratch scratch(st);
  NB_TRY(scratch.alloc(parts.bytes));
  char *base = static_cast<char *>(scratch.p);
  r.partial = reinterpret_cast<float2 *>(base + at_partial);
  r.target = reinterpret_cast<float *>(base + at_target);
  Operand ox, ow;
  NB_TRY(make_operand(x, rows, size, base + at_x, ox, st));
  NB_TRY(make_operand(w, size, classes, base + at_w, ow, st));
  Products prob{};
  prob.count = 1;
  prob.bias = bias;
  prob.rows = r;
  prob.p[0].M = (int)rows, prob.p[0].N = (int)classes, prob.p[0].kblocks = kblocks, prob.p[0].b_mn = 1;
  NB_TRY((pair ? launch_loss_gemm<T, true, Out::kSums> : launch_loss_gemm<T, false, Out::kSums>)(prob, &ox, &ow, st));
  NB_CUDA(launch_dependent(loss_rows_kernel, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, r, rows, loss, stat));
  return NB200_OK;
}

template <typename T>
int backward_tensor(const T *x, const T *w, const T *bias, LossRows r, T *dx, T *dw, T *db, int64_t rows, int64_t size,
                    int64_t classes, const bool accum[3], cudaStream_t st) {
  constexpr bool kF32 = std::is_same<T, float>::value;
  constexpr int kPlanes = kF32 ? 3 : 1;
  using G = std::conditional_t<kF32, __nv_bfloat16, T>;
  // A piece's G is 2^26 values, 128 MB in 16 bits: large enough that the tiles of its products end in one round of few
  // idle SMs, and read from L2 for the most part.
  int64_t piece = std::max<int64_t>(1024, (int64_t)(1 << 26) / kPlanes / rows);
  const int64_t count = (classes + piece - 1) / piece;
  piece = up((classes + count - 1) / count, 256);
  const bool pieces = piece < classes;
  // Few tiles of dx with a long K: its classes in up to 16 parts, each with sums of its own that round_kernel adds up.
  const int64_t size_blocks = (size + 63) / 64, row_blocks = (rows + 63) / 64, piece_blocks = (std::min(piece, classes) + 63) / 64;
  const bool pair_grad = pays_pairs({{rows, piece, size_blocks}});
  const bool pair = pays_pairs({{dw ? size : 0, piece, row_blocks}, {dx ? rows : 0, size, piece_blocks}});
  int splits = 1;
  if (dx) {
    const int64_t tiles = ((rows + (pair ? 255 : 127)) / (pair ? 256 : 128)) * ((size + (pair ? 255 : 63)) / (pair ? 256 : 64));
    const int64_t units = pair ? sm_count() / 2 : sm_count();
    while (splits < 16 && tiles * splits * 2 <= units && piece_blocks >= 8 * splits)
      splits *= 2;
  }
  const int split_blocks = (int)((piece_blocks + splits - 1) / splits);
  splits = (int)((piece_blocks + split_blocks - 1) / split_blocks); // no empty part (a last, smaller piece may leave some)
  const bool direct = splits == 1 && (!pieces || (kF32 && !accum[0])); // dx without sums of its own
  Parts parts;
  const size_t at_x = parts.take(operand_bytes(x, rows, size)), at_w = parts.take(operand_bytes(w, size, classes));
  const size_t at_g = parts.take((size_t)kPlanes * rows * piece * 2), at_scale = parts.take(12);
  const size_t at_dx = parts.take(dx && !direct ? (size_t)splits * rows * size * 4 : 0);
  AsyncScratch scratch(st);
  NB_TRY(scratch.alloc(parts.bytes));
  char *base = static_cast<char *>(scratch.p);
  float *dx32 = reinterpret_cast<float *>(base + at_dx);
  Operand ox, ow;
  NB_TRY(make_operand(x, rows, size, base + at_x, ox, st));
  NB_TRY(make_operand(w, size, classes, base + at_w, ow, st));
  float *scale = reinterpret_cast<float *>(base + at_scale);
  NB_CUDA(launch_dependent(gradient_scale_kernel, dim3(1), dim3(1024), 0, st, r, rows,
                           std::is_same<T, __half>::value ? 16384.0f : 1.0f, scale));
  r.scale = scale;
  for (int64_t c0 = 0; c0 < classes; c0 += piece) {
    const int64_t n = std::min(piece, classes - c0);
    const Operand og{base + at_g, rows, n, piece, kPlanes}, owc = columns(ow, c0, n);
    Products prob{};
    prob.count = 1;
    prob.bias = bias;
    prob.class0 = (int)c0;
    prob.rows = r;
    Product &l = prob.p[0];
    l.M = (int)rows, l.N = (int)n, l.kblocks = (int)size_blocks, l.b_mn = 1;
    l.out = base + at_g, l.ldo = piece, l.stride = rows * piece;
    NB_TRY((pair_grad ? launch_loss_gemm<T, true, Out::kGrad> : launch_loss_gemm<T, false, Out::kGrad>)(prob, &ox, &owc, st));
    Operand a[2], b[2];
    prob.count = 0;
    if (dw) {
      Product &p = prob.p[prob.count];
      p = Product{};
      p.M = (int)size, p.N = (int)n, p.kblocks = (int)row_blocks, p.a_mn = p.b_mn = 1;
      p.out = dw + c0, p.ldo = classes, p.accum = accum[1];
      p.vec = classes * sizeof(T) % 16 == 0 && aligned16(dw);
      a[prob.count] = ox, b[prob.count++] = og;
    }
    if (dx) {
      Product &p = prob.p[prob.count];
      p = Product{};
      p.M = (int)rows, p.N = (int)size, p.kblocks = (int)((n + 63) / 64), p.ldo = size;
      p.splits = (p.kblocks + split_blocks - 1) / split_blocks, p.split_blocks = split_blocks, p.stride = rows * size;
      p.out = direct ? static_cast<void *>(dx) : dx32, p.out_f32 = !direct;
      p.accum = c0 > 0 || (direct && accum[0]);
      p.vec = size * (p.out_f32 ? 4 : sizeof(T)) % 16 == 0 && aligned16(p.out);
      a[prob.count] = og, b[prob.count++] = owc;
    }
    if (prob.count)
      NB_TRY((pair ? launch_loss_gemm<T, true, Out::kStore> : launch_loss_gemm<T, false, Out::kStore>)(prob, a, b, st));
    if (db)
      NB_CUDA(launch_dependent(column_sums_kernel<G, T>, dim3((unsigned)((n + 31) / 32)), dim3(512), 0, st,
                               reinterpret_cast<const G *>(base + at_g), kPlanes, rows, n, piece, r.scale, db + c0, accum[2]));
  }
  if (dx && !direct)
    NB_CUDA(launch_dependent(round_kernel<T>, dim3((unsigned)std::min<int64_t>((rows * size + 255) / 256, 8 * sm_count())),
                             dim3(256), 0, st, (const float *)dx32, splits, dx, rows * size, accum[0]));
  return NB200_OK;
}

template <typename T>
int forward(const T *x, const T *w, const T *bias, LossRows r, float *loss, float2 *stat, int64_t rows, int64_t size,
            cudaStream_t st) {
  if (rows > kFewRows)
    return forward_tensor<T>(x, w, bias, r, loss, stat, rows, size, r.classes, st);
  const bool vec = r.classes % kPackOf<T> == 0 && aligned16(w);
  const int64_t columns = vec ? few_lanes<T, kPackOf<T>>() * kPackOf<T> : 32;
  r.tiles = (int)((r.classes + columns - 1) / columns);
  AsyncScratch scratch(st);
  NB_TRY(scratch.alloc((size_t)rows * r.tiles * 8 + (size_t)rows * 4));
  r.partial = static_cast<float2 *>(scratch.p);
  r.target = reinterpret_cast<float *>(r.partial + rows * r.tiles);
  NB_TRY(few_variant<T>(rows, vec, [&](auto n, auto v) {
    return few_logits<T, decltype(n)::value, decltype(v)::value>(x, w, bias, r, (int)rows, size, nullptr, 0, st);
  }));
  NB_CUDA(launch_dependent(loss_rows_kernel, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, r, rows, loss, stat));
  return NB200_OK;
}

template <typename T>
int backward(const T *x, const T *w, const T *bias, LossRows r, T *dx, T *dw, T *db, int64_t rows, int64_t size,
             const bool accum[3], cudaStream_t st) {
  if (rows > kFewRows)
    return backward_tensor<T>(x, w, bias, r, dx, dw, db, rows, size, r.classes, accum, st);
  const int64_t classes = r.classes, ldg = up(classes, 4);
  AsyncScratch scratch(st);
  NB_TRY(scratch.alloc((size_t)rows * ldg * 4));
  float *g = static_cast<float *>(scratch.p);
  const bool vec = classes % kPackOf<T> == 0 && aligned16(w);
  NB_TRY(few_variant<T>(rows, vec, [&](auto n, auto v) {
    return few_logits<T, decltype(n)::value, decltype(v)::value>(x, w, bias, r, (int)rows, size, g, ldg, st);
  }));
  if (dx || dw) {
    const bool keep = (size_t)size * classes * sizeof(T) <= kKeepBytes;
    NB_TRY(few_variant<T>(rows, vec && aligned16(dw), [&](auto n, auto v) -> int {
      NB_CUDA(launch_dependent(few_grads_kernel<T, decltype(n)::value, decltype(v)::value>,
                               dim3((unsigned)((size + kFewH - 1) / kFewH)), dim3(kFewGradThreads), 0, st, x, w,
                               (const float *)g, ldg, dx, dw, (int)rows, size, classes, accum[0], accum[1], keep));
      return NB200_OK;
    }));
  }
  if (db)
    NB_CUDA(launch_dependent(column_sums_kernel<float, T>, dim3((unsigned)((classes + 31) / 32)), dim3(512), 0, st,
                             (const float *)g, 1, rows, classes, ldg, (const float *)nullptr, db, accum[2]));
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
    LossRows r{};
    r.label = label, r.label_bytes = label_bytes, r.classes = classes;
    return forward<T>(static_cast<const T *>(x), static_cast<const T *>(w), static_cast<const T *>(bias), r, loss,
                      reinterpret_cast<float2 *>(stat), rows, size, as_stream(stream));
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
    LossRows r{};
    r.label = label, r.label_bytes = label_bytes, r.classes = classes;
    r.stat = reinterpret_cast<const float2 *>(stat), r.dloss = dloss;
    return backward<T>(static_cast<const T *>(x), static_cast<const T *>(w), static_cast<const T *>(bias), r,
                       static_cast<T *>(dx), static_cast<T *>(dw), static_cast<T *>(db), rows, size, accum, as_stream(stream));
  });
}
