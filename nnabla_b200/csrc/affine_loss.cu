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

namespace nb200 {
namespace {

// The rows' loss and statistics from the tiles' maxima and sums: `share` of a block's eight warps a row (all of them where rows
// are few and their tiles many: 3408 of nine rows took one warp each 17 us).
__global__ void __launch_bounds__(256) loss_rows_kernel(LossRows rows, int64_t count, int share, float *__restrict__ loss,
                                                        float2 *__restrict__ stat) {
  __shared__ float2 parts[8];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = warp % share;
  const int64_t row = (int64_t)blockIdx.x * (8 / share) + warp / share;
  MaxSum t{-INFINITY, 0.0f};
  if (row < count)
#pragma unroll 4
    for (int i = mine * 32 + lane; i < rows.tiles; i += 32 * share) {
      const float2 p = rows.partial[row * rows.tiles + i];
      t = join(t, MaxSum{p.x, p.y}, kLog2e);
    }
  t = warp_join(t, kLog2e);
  if (share > 1) {
    if (lane == 0)
      parts[warp] = make_float2(t.m, t.s);
    __syncthreads();
    if (mine == 0)
      for (int w = 1; w < share; ++w)
        t = join(t, MaxSum{parts[warp + w].x, parts[warp + w].y}, kLog2e);
  }
  if (lane == 0 && mine == 0 && row < count) {
    const int64_t label = rows.label_of(row);
    const float log_sum = log2f(t.s) * kLn2;
    stat[row] = make_float2(t.m, log_sum);
    loss[row] = label < 0 ? 0.0f : label >= rows.classes ? NAN : (t.m - rows.target[row]) + log_sum;
  }
}
int loss_rows(const LossRows &r, int64_t count, float *loss, float2 *stat, cudaStream_t st) {
  const int share = r.tiles > 64 && count <= 8 * sm_count() ? 8 : 1;
  NB_CUDA(launch_dependent(loss_rows_kernel, dim3((unsigned)((count * share + 7) / 8)), dim3(256), 0, st, r, count, share, loss,
                           stat));
  return NB200_OK;
}

// Column sums of G, [planes][rows][ld]: a thread eight (fp32: four) neighbouring columns, a block's eight warps its slab of
// rows in turn; part[slab][ldp].
template <typename G>
__global__ void __launch_bounds__(256) column_sums_kernel(const G *__restrict__ g, int64_t all_rows, int64_t slab,
                                                          int64_t columns, int64_t ld, float *__restrict__ part, int64_t ldp) {
  constexpr int V = kPackOf<G>;
  __shared__ float sums[8][32 * V];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c0 = (int64_t)blockIdx.x * 32 * V, c = c0 + lane * V, r0 = blockIdx.y * slab;
  const int64_t r1 = r0 + slab < all_rows ? r0 + slab : all_rows;
  float s[V];
#pragma unroll
  for (int j = 0; j < V; ++j)
    s[j] = 0.0f;
  if (c < columns) // (ld is a multiple of V and G is as wide)
#pragma unroll 4
    for (int64_t r = r0 + warp; r < r1; r += 8) {
      const Pack<G, V> p = load_pack<G, V>(g + r * ld + c);
#pragma unroll
      for (int j = 0; j < V; ++j)
        s[j] += p.f(j);
    }
#pragma unroll
  for (int j = 0; j < V; ++j)
    sums[warp][lane * V + j] = s[j];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * V; i += 256) {
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w)
      t += sums[w][i];
    if (c0 + i < ldp)
      part[blockIdx.y * ldp + c0 + i] = t;
  }
}

// to [rows][ldt] (+)= scale[2] (scale NULL: 1) * the sum, in order, of `parts` matrices [rows][ldf], `stride` apart.
// V columns a thread.
template <typename T, int V>
__global__ void __launch_bounds__(256) add_parts_kernel(const float *__restrict__ from, int parts, int64_t stride, int64_t rows,
                                                        int64_t cols, int64_t ldf, const float *scale, T *to, int64_t ldt,
                                                        bool accum) {
  pdl_wait();
  pdl_trigger();
  const int64_t packs = (cols + V - 1) / V;
  const float times = scale ? scale[2] : 1.0f;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * packs; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / packs, c = (i - r * packs) * V;
    float s[V];
#pragma unroll
    for (int j = 0; j < V; ++j)
      s[j] = 0.0f;
#pragma unroll 8
    for (int p = 0; p < parts; ++p) {
      const Pack<float, V> f = load_pack<float, V>(from + p * stride + r * ldf + c);
#pragma unroll
      for (int j = 0; j < V; ++j)
        s[j] += f.f(j);
    }
    T *t = to + r * ldt + c;
    Pack<T, V> old;
    if (accum)
      old = load_pack<T, V>(t);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      s[j] *= times;
      if (accum)
        s[j] += old.f(j);
    }
    store_pack<T, V>(t, s);
  }
}
template <typename T>
int add_parts(const float *from, int parts, int64_t stride, int64_t rows, int64_t cols, int64_t ldf, const float *scale, T *to,
              int64_t ldt, bool accum, cudaStream_t st) {
  const bool vec = cols % 4 == 0 && stride % 4 == 0 && ldf % 4 == 0 && ldt % 4 == 0 && aligned16(from) &&
                   (reinterpret_cast<uintptr_t>(to) & (4 * sizeof(T) - 1)) == 0;
  const int64_t items = rows * ((cols + (vec ? 3 : 0)) / (vec ? 4 : 1));
  const dim3 grid((unsigned)std::max<int64_t>(1, std::min<int64_t>((items + 255) / 256, 16 * sm_count())));
  NB_CUDA(launch_dependent(vec ? add_parts_kernel<T, 4> : add_parts_kernel<T, 1>, grid, dim3(256), 0, st, from, parts, stride,
                           rows, cols, ldf, scale, to, ldt, accum));
  return NB200_OK;
}

// db (+)= the column sums of G [planes * rows][ld], of which `part`, room floats of scratch, holds a row of ld sums for each slab.
template <typename G, typename T>
int column_sums(const G *g, int64_t all_rows, Slabs slabs, int64_t columns, int64_t ld, float *part, int64_t room,
                const float *scale, T *db, bool accum, cudaStream_t st) {
  static_assert(32 * kPackOf<G> == kSumColumns, "a block's columns");
  NB_CHECK(slabs.count * ld <= room && slabs.count * slabs.rows >= all_rows, NB200_EVALUE, "sums of %lld slabs of %lld classes",
           (long long)slabs.count, (long long)ld);
  const int64_t wide = (columns + kSumColumns - 1) / kSumColumns;
  NB_CUDA(launch_dependent(column_sums_kernel<G>, dim3((unsigned)wide, (unsigned)slabs.count), dim3(256), 0, st, g, all_rows,
                           slabs.rows, columns, ld, part, ld));
  return add_parts<T>(part, (int)slabs.count, ld, 1, columns, ld, scale, db, 0, accum, st);
}

// What the tensor-core products need before they start, in one launch: up to two matrices laid out as operands (fp32: three
// bf16 pieces; 16 bits: rows at a pitch that a TMA copy can read), and the scale of G.
struct Layout {
  const void *from; // NULL: the matrix is an operand as it lies
  void *to;
  int64_t rows, cols, pitch, packs; // packs: rows * pitch / 8
};
struct Preparation {
  Layout m[2];
  unsigned blocks[2]; // blocks of 256 threads for each, eight values a thread and step
  LossRows rows;      // G's scale, by one more block where scale is not NULL
  int64_t count;
  float times;
  float *scale;
};

// scale = {the largest finite |dloss| of a row whose label is a class, 2^e, their quotient}: what G is kept relative to (the other
// rows of G are 0, infinite or NaN whatever it is, and no gradient of theirs changes how another row is rounded). With the
// largest taken out, the gradient of a mean, the same in every row, is no rounded factor of G: at the label G is -1 + p. e is 14
// for an fp16 G, which so has eleven bits down to 2^-28 of the largest gradient, and 0 for the others.
__device__ void gradient_scale(const Preparation &p) {
  __shared__ float tops[8];
  float top = 0.0f;
#pragma unroll 8
  for (int64_t r = threadIdx.x; r < p.count; r += 256) {
    const int64_t label = p.rows.label_of(r);
    const float d = fabsf(p.rows.dloss[r]);
    top = fmaxf(top, label >= 0 && label < p.rows.classes && d < INFINITY ? d : 0.0f);
  }
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0)
    tops[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < 8; ++w)
      top = fmaxf(top, tops[w]);
    const bool plain = !(top >= 1.17549435e-38f); // none, or none that can be divided by
    p.scale[0] = plain ? 1.0f : top;
    p.scale[1] = p.times;
    p.scale[2] = (plain ? 1.0f : top) / p.times;
  }
}

template <typename T> __global__ void __launch_bounds__(256) loss_prepare_kernel(const __grid_constant__ Preparation p) {
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x == p.blocks[0] + p.blocks[1]) {
    gradient_scale(p);
    return;
  }
  const int which = blockIdx.x < p.blocks[0] ? 0 : 1;
  const Layout &m = p.m[which];
  const T *from = static_cast<const T *>(m.from);
  const bool vec = std::is_same<T, float>::value && m.cols % 4 == 0 && (reinterpret_cast<uintptr_t>(from) & 15) == 0;
  const int64_t per_row = m.pitch / 8, step = (int64_t)p.blocks[which] * 256;
  for (int64_t i = (int64_t)(blockIdx.x - (which ? p.blocks[0] : 0)) * 256 + threadIdx.x; i < m.packs; i += step) {
    const int64_t r = i / per_row, c = (i - r * per_row) * 8;
    const T *src = from + r * m.cols + c;
    Pack<T, 8> v;
    if (vec && c + 8 <= m.cols) {
      v = load_pack<T, 8>(src);
    } else {
      v.clear();
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < m.cols)
          v.set(j, src[j]);
    }
    if constexpr (std::is_same<T, float>::value) {
      __nv_bfloat16 *to = static_cast<__nv_bfloat16 *>(m.to) + r * m.pitch + c;
      float left[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        left[j] = v.f(j);
#pragma unroll
      for (int pl = 0; pl < 3; ++pl) {
        const Pack<__nv_bfloat16, 8> h = round_pack<__nv_bfloat16, 8>(left);
        *reinterpret_cast<Pack<__nv_bfloat16, 8> *>(to + pl * m.rows * m.pitch) = h;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          left[j] = __fsub_rn(left[j], h.f(j));
      }
    } else {
      *reinterpret_cast<Pack<T, 8> *>(static_cast<T *>(m.to) + r * m.pitch + c) = v;
    }
  }
}

// A matrix as an operand of the tensor-core products: as it lies, or laid out anew in operand_bytes() of scratch.
template <typename T> size_t operand_bytes(const T *p, int64_t rows, int64_t cols) {
  if (std::is_same<T, float>::value)
    return (size_t)3 * rows * up(cols, 64) * 2;
  return cols % 8 == 0 && aligned16(p) ? 0 : (size_t)rows * up(cols, 8) * 2;
}
template <typename T> Operand operand(const T *p, int64_t rows, int64_t cols, void *scratch, Layout &layout) {
  constexpr bool kF32 = std::is_same<T, float>::value;
  Operand o{scratch, rows, cols, up(cols, kF32 ? 64 : 8), kF32 ? 3 : 1, rows};
  layout = Layout{};
  if (operand_bytes(p, rows, cols) == 0)
    o.p = p;
  else
    layout = Layout{p, scratch, rows, cols, o.pitch, rows * o.pitch / 8};
  return o;
}
template <typename T> int prepare(Preparation &p, cudaStream_t st) {
  for (int i = 0; i < 2; ++i)
    p.blocks[i] = p.m[i].from ? (unsigned)std::min<int64_t>((p.m[i].packs + 255) / 256, 32 * sm_count()) : 0;
  const unsigned blocks = p.blocks[0] + p.blocks[1] + (p.scale ? 1 : 0);
  if (blocks)
    NB_CUDA(launch_dependent(loss_prepare_kernel<T>, dim3(blocks), dim3(256), 0, st, p));
  return NB200_OK;
}
Operand columns(Operand o, int64_t c0, int64_t n) {
  o.p = static_cast<const char *>(o.p) + 2 * c0;
  o.cols = n;
  return o;
}

template <typename T>
int forward_tensor(const T *x, const T *w, const T *bias, LossRows r, float *loss, float2 *stat, int64_t rows, int64_t size,
                   int64_t classes, cudaStream_t st) {
  const int kblocks = (int)((size + 63) / 64);
  const bool pair = pays_pairs({{rows, classes, kblocks}}, sm_count());
  const bool split = std::is_same<T, float>::value && loss_splits(rows, size, classes);
  r.tiles = split ? (int)((classes + kSplitTile - 1) / kSplitTile) * 2 : loss_sum_tiles<T>(classes, kblocks, pair);
  // so many rows at a time that their maxima and sums are 64 MB (the largest head in use: 8192 rows of 128000 classes)
  const int64_t slab = std::min(rows, std::max<int64_t>(256, (1 << 23) / r.tiles / 256 * 256));
  Parts parts;
  const size_t at_x = parts.take(operand_bytes(x, rows, size)), at_w = parts.take(split ? 0 : operand_bytes(w, size, classes));
  const size_t at_partial = parts.take((size_t)slab * r.tiles * 8), at_target = parts.take((size_t)slab * 4);
  AsyncScratch scratch(st);
  NB_TRY(scratch.alloc(parts.bytes));
  char *base = static_cast<char *>(scratch.p);
  r.partial = reinterpret_cast<float2 *>(base + at_partial);
  r.target = reinterpret_cast<float *>(base + at_target);
  Preparation pre{};
  const Operand ox = operand(x, rows, size, base + at_x, pre.m[0]), ow = operand(w, size, classes, base + at_w, pre.m[1]);
  if (split)
    pre.m[1] = Layout{};
  NB_TRY(prepare<T>(pre, st));
  const char *label = static_cast<const char *>(r.label);
  for (int64_t r0 = 0; r0 < rows; r0 += slab) {
    const int64_t n = std::min(slab, rows - r0);
    Operand part = ox; // (its planes stay as far apart)
    part.p = static_cast<const char *>(ox.p) + 2 * r0 * ox.pitch;
    part.rows = n;
    r.label = label + r0 * r.label_bytes;
    Products prob{};
    prob.count = 1;
    prob.bias = bias;
    prob.rows = r;
    prob.p[0].M = (int)n, prob.p[0].N = (int)classes, prob.p[0].K = (int)size, prob.p[0].kblocks = kblocks, prob.p[0].b_mn = 1;
    if constexpr (std::is_same<T, float>::value)
      if (split) {
        NB_TRY(run_split_gemm<Out::kSums>(prob, part, w, size, classes, classes, st));
        NB_TRY(loss_rows(r, n, loss + r0, stat + r0, st));
        continue;
      }
    NB_TRY((run_loss_gemm<T, Out::kSums>(pair, prob, &part, &ow, st)));
    NB_TRY(loss_rows(r, n, loss + r0, stat + r0, st));
  }
  return NB200_OK;
}

template <typename T>
int backward_tensor(const T *x, const T *w, const T *bias, LossRows r, T *dx, T *dw, T *db, int64_t rows, int64_t size,
                    int64_t classes, const bool accum[3], cudaStream_t st) {
  constexpr bool kF32 = std::is_same<T, float>::value;
  constexpr int kPlanes = kF32 ? 3 : 1;
  using G = std::conditional_t<kF32, __nv_bfloat16, T>;
  const bool split = kF32 && loss_splits(rows, size, classes);
  const HeadGradients plan(rows, size, classes, kF32, dx, dw, db, accum[0], operand_bytes(x, rows, size),
                           split ? 0 : operand_bytes(w, size, classes), sm_count());
  const int64_t piece = plan.piece, ld_dx = plan.ld_dx;
  const bool direct = plan.direct;
  AsyncScratch scratch(st);
  NB_TRY(scratch.alloc(plan.bytes));
  char *base = static_cast<char *>(scratch.p);
  float *dx32 = reinterpret_cast<float *>(base + plan.at_dx), *dw32 = reinterpret_cast<float *>(base + plan.at_dw);
  float *scale = reinterpret_cast<float *>(base + plan.at_scale);
  Preparation pre{};
  const Operand ox = operand(x, rows, size, base + plan.at_x, pre.m[0]), ow = operand(w, size, classes, base + plan.at_w, pre.m[1]);
  if (split)
    pre.m[1] = Layout{};
  pre.rows = r, pre.count = rows, pre.scale = scale, pre.times = std::is_same<T, __half>::value ? 16384.0f : 1.0f;
  NB_TRY(prepare<T>(pre, st));
  r.scale = scale;
  for (int64_t c0 = 0; c0 < classes; c0 += piece) {
    const int64_t n = plan.classes_at(c0);
    const Operand og{base + plan.at_g, rows, n, piece, kPlanes, rows}, owc = columns(ow, c0, n);
    Products prob{};
    prob.count = 1;
    prob.bias = bias;
    prob.class0 = (int)c0;
    prob.rows = r;
    Product &l = prob.p[0];
    l.M = (int)rows, l.N = (int)n, l.K = (int)size, l.kblocks = (int)((size + 63) / 64), l.b_mn = 1;
    l.out = base + plan.at_g, l.ldo = piece, l.stride = rows * piece;
    if constexpr (kF32) {
      if (split)
        NB_TRY(run_split_gemm<Out::kGrad>(prob, ox, w + c0, size, n, classes, st));
      else
        NB_TRY((run_loss_gemm<T, Out::kGrad>(plan.pair_grad, prob, &ox, &owc, st)));
    } else {
      NB_TRY((run_loss_gemm<T, Out::kGrad>(plan.pair_grad, prob, &ox, &owc, st)));
    }
    Operand a[2], b[2];
    prob.count = 0;
    if (dw) {
      Product &p = prob.p[prob.count];
      p = Product{};
      p.M = (int)size, p.N = (int)n, p.K = (int)rows, p.kblocks = (int)((rows + 63) / 64), p.a_mn = p.b_mn = 1;
      if (plan.dw_splits > 1) {
        p.splits = plan.dw_splits, p.split_blocks = plan.dw_blocks, p.stride = size * piece;
        p.out = dw32, p.ldo = piece, p.out_f32 = 1, p.vec = 1;
      } else {
        p.out = dw + c0, p.ldo = classes, p.accum = accum[1];
        p.vec = classes * sizeof(T) % 16 == 0 && aligned16(dw);
      }
      a[prob.count] = ox, b[prob.count++] = og;
    }
    if (dx) {
      Product &p = prob.p[prob.count];
      p = Product{};
      p.M = (int)rows, p.N = (int)size, p.K = (int)n, p.kblocks = (int)((n + 63) / 64), p.ldo = direct ? size : ld_dx;
      p.splits = (p.kblocks + plan.dx_blocks - 1) / plan.dx_blocks, p.split_blocks = plan.dx_blocks, p.stride = rows * ld_dx;
      p.out = direct ? static_cast<void *>(dx) : dx32, p.out_f32 = !direct;
      p.accum = c0 > 0 || (direct && accum[0]);
      p.vec = p.ldo * (p.out_f32 ? 4 : sizeof(T)) % 16 == 0 && aligned16(p.out);
      a[prob.count] = og, b[prob.count++] = owc;
    }
    if constexpr (kF32)
      if (split && dx) { // dx for itself, the last of the products
        Products one = prob;
        one.count = 1;
        one.p[0] = prob.p[--prob.count];
        NB_TRY(run_split_gemm<Out::kStore>(one, og, w + c0, size, n, classes, st));
      }
    if (!kF32 && prob.count == 2 && loss_is_long<T>(plan.dx_blocks) != loss_is_long<T>(plan.dw_blocks)) {
      // (of two forms of the kernel: together both would take the one with eight epilogue warps)
      for (int i = 0; i < 2; ++i) {
        Products one = prob;
        one.count = 1;
        one.p[0] = prob.p[i];
        const Product &p = one.p[0];
        const int64_t blocks = p.splits > 1 ? p.split_blocks : p.kblocks;
        NB_TRY((run_loss_gemm<T, Out::kStore>(pays_pairs({{p.M, p.N, blocks, std::max(1, p.splits)}}, sm_count()), one, a + i,
                                               b + i, st)));
      }
    } else if (prob.count) {
      NB_TRY((run_loss_gemm<T, Out::kStore>(plan.pair, prob, a, b, st)));
    }
    if (dw && plan.dw_splits > 1)
      NB_TRY(add_parts<T>(dw32, plan.dw_splits, size * piece, size, n, piece, nullptr, dw + c0, classes, accum[1], st));
    if (db)
      NB_TRY((column_sums<G, T>(reinterpret_cast<const G *>(base + plan.at_g), kPlanes * rows, plan.db, n, piece,
                                reinterpret_cast<float *>(base + plan.at_db), (int64_t)(plan.bytes - plan.at_db) / 4, scale,
                                db + c0, accum[2], st)));
  }
  if (dx && !direct)
    NB_TRY(add_parts<T>(dx32, plan.dx_splits, rows * ld_dx, rows, size, ld_dx, nullptr, dx, size, accum[0], st));
  return NB200_OK;
}

template <typename T>
int forward(const T *x, const T *w, const T *bias, LossRows r, float *loss, float2 *stat, int64_t rows, int64_t size,
            cudaStream_t st) {
  if (rows > kFewRows)
    return forward_tensor<T>(x, w, bias, r, loss, stat, rows, size, r.classes, st);
  const bool aligned = few_aligned(w, r.classes);
  int columns = 0;
  NB_TRY(few_variant(rows, [&](auto n) -> int {
    constexpr int R = decltype(n)::value;
    columns = aligned ? few_columns<T, R, false>() : few_columns<T, R, true>();
    return NB200_OK;
  }));
  r.tiles = (int)((r.classes + columns - 1) / columns);
  AsyncScratch scratch(st);
  NB_TRY(scratch.alloc((size_t)rows * r.tiles * 8 + (size_t)rows * 4));
  r.partial = static_cast<float2 *>(scratch.p);
  r.target = reinterpret_cast<float *>(r.partial + rows * r.tiles);
  NB_TRY(few_variant(rows, [&](auto n) {
    constexpr int R = decltype(n)::value;
    return (aligned ? few_logits<T, R, false> : few_logits<T, R, true>)(x, w, bias, r, (int)rows, size, nullptr, 0, st);
  }));
  return loss_rows(r, rows, loss, stat, st);
}

template <typename T>
int backward(const T *x, const T *w, const T *bias, LossRows r, T *dx, T *dw, T *db, int64_t rows, int64_t size,
             const bool accum[3], cudaStream_t st) {
  if (rows > kFewRows)
    return backward_tensor<T>(x, w, bias, r, dx, dw, db, rows, size, r.classes, accum, st);
  const int64_t classes = r.classes, ldg = up(classes, 4);
  const bool aligned = few_aligned(w, classes);
  // Both gradients in one pass, unless rows of W and dW begin differently far behind a 16-byte boundary.
  const bool alike = !dx || !dw || ((reinterpret_cast<uintptr_t>(w) ^ reinterpret_cast<uintptr_t>(dw)) & 15) == 0;
  const FewGradients plan(size, classes, kPackOf<T>, !few_aligned(dx ? w : dw, classes), sm_count());
  Parts parts;
  const size_t at_g = parts.take((size_t)rows * ldg * 4), at_dx = parts.take(dx ? (size_t)plan.columns * rows * size * 4 : 0);
  AsyncScratch scratch(st);
  NB_TRY(scratch.alloc(parts.bytes));
  char *base = static_cast<char *>(scratch.p);
  float *g = reinterpret_cast<float *>(base + at_g), *dx32 = reinterpret_cast<float *>(base + at_dx);
  NB_TRY(few_variant(rows, [&](auto n) {
    constexpr int R = decltype(n)::value;
    return (aligned ? few_logits<T, R, false> : few_logits<T, R, true>)(x, w, bias, r, (int)rows, size, g, ldg, st);
  }));
  if (dx || dw) {
    const bool keep = (size_t)size * classes * sizeof(T) <= kKeepBytes;
    auto grads = [&](const FewGradients &p, T *to_dx, T *to_dw) {
      return few_variant(rows, [&](auto n) -> int {
        constexpr int R = decltype(n)::value;
        auto kernel = few_aligned(to_dx ? w : to_dw, classes) ? few_grads_kernel<T, R, false> : few_grads_kernel<T, R, true>;
        NB_CUDA(launch_dependent(kernel, dim3((unsigned)p.columns, (unsigned)p.blocks), dim3(kFewGradThreads), 0, st, x, w,
                                 (const float *)g, ldg, to_dx != nullptr, to_dw, dx32, (int)rows, size, p.slab, classes, accum[1],
                                 keep));
        return NB200_OK;
      });
    };
    NB_TRY(grads(plan, dx, alike ? dw : nullptr));
    if (!alike)
      NB_TRY(grads(FewGradients(size, classes, kPackOf<T>, !few_aligned(dw, classes), sm_count()), nullptr, dw));
    if (dx)
      NB_TRY(add_parts<T>(dx32, (int)plan.columns, rows * size, 1, rows * size, rows * size, nullptr, dx, rows * size, accum[0], st));
  }
  if (db)
    NB_TRY(add_parts<T>(g, (int)rows, ldg, 1, classes, ldg, nullptr, db, classes, accum[2], st));
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
