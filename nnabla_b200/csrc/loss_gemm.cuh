// The products of a classifying head on tcgen05: l = x W, dx = G W^T, dW = x^T G, each from the operands as they lie.
//
// Clusters of two CTAs make a 256 x BN tile (cta_group::2): each loads its own 128 rows of A and its own BN / 2 columns of B
// by TMA, the leader issues the MMAs, both drain their 128 accumulator rows. W [inputs, classes] has its classes in
// neighbouring memory, so in l = x W, and for both operands of dW, the rows of memory run along K: those operands are read as
// MN-major ones, stored as chunks of 64 rows (K) x 128 bytes (bit 15 / 16 of the instruction descriptor; the leading byte
// offset leads from one chunk of 64 columns to the next). Nothing is transposed.
//
// PL planes an operand: 1 (bf16 or fp16 as it is) or 3 (the bf16 pieces of an fp32 tensor; the six products that matter at
// fp32 resolution). The tensor core's additions truncate: every 96 MMA steps the accumulator is added up in fp32 registers
// (gemm.cuh).
//
// What becomes of a tile, by the epilogue:
//   kSums   of each row and half of a tile's column chunks, the maximum and the sum of the exponentials; the label's logit
//   kGrad   G, in 16 bits (fp32: three bf16 planes)
//   kStore  the product itself, two products (dx and dW of a piece of the classes) in one launch: with one after the other,
//           each would end in a round of tiles that leaves SMs idle
#pragma once
#include "gemm2.cuh"
#include "softmax_sums.cuh"

namespace nb200 {

// A row's label and, for the backward pass, its statistics and the gradient that arrives.
struct LossRows {
  const void *label; // label_bytes each
  int label_bytes;
  int64_t classes;
  const float2 *stat;
  const float *dloss;
  const float *scale; // G is kept relative to dloss = scale[0] and times scale[1]; scale[2] = scale[0] / scale[1]
  float2 *partial;    // kSums: [rows][tiles]
  float *target;      // [rows], the label's logit
  int tiles;
  __device__ __forceinline__ int64_t label_of(int64_t row) const {
    return label_bytes == 8 ? static_cast<const int64_t *>(label)[row] : (int64_t) static_cast<const int32_t *>(label)[row];
  }
};

enum class Out { kSums, kGrad, kStore };

constexpr int kMaxProducts = 2;
struct Product {
  int M, N, kblocks, m_tiles, n_tiles;
  int a_mn, b_mn; // memory rows run along K
  // kStore: out [M][ldo] (+)= scale[2] * D (+ base, fp32); kGrad: out is G [planes][M][ldo]
  void *out;
  const float *base;
  int64_t ldo, plane;
  int out_f32, accum;
};
struct Products {
  Product p[kMaxProducts];
  int count;
  int chunk; // K blocks accumulated in tensor memory
  int class0; // kSums, kGrad: the class of the first column
  const void *bias;
  LossRows rows;
};

// stages of the operands' ring
template <int PL, int BN> constexpr int loss_stages() { return PL == 1 ? (BN == 256 ? 6 : 8) : 2; }
template <int PL, int BN> constexpr size_t loss_smem_bytes() {
  return (size_t)loss_stages<PL, BN>() * PL * (kTileM + BN / 2) * kRowBytes + kEpilogueStageBytes +
         (2 * loss_stages<PL, BN>() + 4) * 8 + 16 + 1024;
}

// T: the operands' type; float means three bf16 planes.
template <typename T, int BN, Out kOut>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    loss_gemm_kernel(const __grid_constant__ CUtensorMap map_a0, const __grid_constant__ CUtensorMap map_b0,
                     const __grid_constant__ CUtensorMap map_a1, const __grid_constant__ CUtensorMap map_b1,
                     const __grid_constant__ Products prob, int *status) {
  constexpr bool kF32 = std::is_same<T, float>::value;
  constexpr int PL = kF32 ? 3 : 1, STAGES = loss_stages<PL, BN>();
  constexpr uint32_t kABytes = kTileM * kRowBytes, kBBytes = (BN / 2) * kRowBytes;
  constexpr uint32_t kStageBytes = PL * (kABytes + kBBytes);
  constexpr uint32_t kChunkBytes = 64 * kRowBytes; // 64 columns x 64 of K of an MN-major operand
  constexpr int kMyChunks = BN / 64;               // column chunks of 32 that an epilogue warp drains
  constexpr uint32_t kTmemCols = 2 * BN;

  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float *stage_out = reinterpret_cast<float *>(smem + STAGES * kStageBytes);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + STAGES * kStageBytes + kEpilogueStageBytes);
  uint64_t *full_bar = bars, *empty_bar = bars + STAGES, *tmem_full = bars + 2 * STAGES, *tmem_empty = tmem_full + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tmem_empty + 2);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank(); // 0 = leader
  const int pair_id = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int tiles0 = prob.p[0].m_tiles * prob.p[0].n_tiles;
  const int num_tiles = tiles0 + (kOut == Out::kStore && prob.count > 1 ? prob.p[1].m_tiles * prob.p[1].n_tiles : 0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      ptx::mbar_init(full_bar + s, 1);
      ptx::mbar_init(empty_bar + s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      ptx::mbar_init(tmem_full + b, 1);
      ptx::mbar_init(tmem_empty + b, 2 * kPairEpilogueWarps);
    }
    *abort_flag = 0;
    ptx::mbar_fence_init();
    ptx::prefetch_tensormap(&map_a0);
    ptx::prefetch_tensormap(&map_b0);
  }
  if (warp == 1) {
    ptx::tmem_alloc_pair(tmem_slot, kTmemCols);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::cluster_sync(); // the peer's barriers are initialised before anything is signalled remotely
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();

  auto gave_up = [&](int code) {
    if (*abort_flag == 0)
      atomicCAS(status, 0, code);
    *abort_flag = 1;
  };
  // the product, first row and first column of a tile; rows vary fastest, so that the tiles in flight share columns of B
  auto decode = [&](int tile, int &m0, int &n0) -> int {
    const int which = kOut == Out::kStore && tile >= tiles0 ? 1 : 0;
    tile -= which ? tiles0 : 0;
    const int mt = prob.p[which].m_tiles;
    n0 = tile / mt * BN;
    m0 = tile % mt * kPairTileM;
    return which;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    if (ptx::elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint64_t keep = ptx::l2_policy_evict_last();
      for (int tile = pair_id; tile < num_tiles && ok; tile += num_pairs) {
        int m0, n0;
        const int which = decode(tile, m0, n0);
        const Product &p = prob.p[which];
        const CUtensorMap *ma = which ? &map_a1 : &map_a0, *mb = which ? &map_b1 : &map_b0;
        m0 += (int)rank * kTileM;
        n0 += (int)rank * (BN / 2);
        for (int kb = 0; kb < p.kblocks; ++kb) {
          if (!ptx::mbar_wait(empty_bar + stage, phase ^ 1u, abort_flag)) {
            gave_up(kStatusProducerTimeout);
            ok = false;
            break;
          }
          uint8_t *st = smem + stage * kStageBytes;
          const uint32_t full = ptx::map_to_cta(ptx::smem_u32(full_bar + stage), 0);
          if (rank == 0)
            ptx::mbar_expect_tx(full_bar + stage, 2 * kStageBytes); // bytes of both CTAs
#pragma unroll
          for (int pl = 0; pl < PL; ++pl) {
            uint8_t *a = st + pl * kABytes, *b = st + PL * kABytes + pl * kBBytes;
            if (p.a_mn) {
#pragma unroll
              for (int j = 0; j < kTileM / 64; ++j)
                ptx::tma_load_3d_pair(a + j * kChunkBytes, ma, full, m0 + 64 * j, kb * 64, pl, keep);
            } else {
              ptx::tma_load_3d_pair(a, ma, full, kb * 64, m0, pl, keep);
            }
            if (p.b_mn) {
#pragma unroll
              for (int j = 0; j < BN / 128; ++j)
                ptx::tma_load_3d_pair(b + j * kChunkBytes, mb, full, n0 + 64 * j, kb * 64, pl, keep);
            } else {
              ptx::tma_load_3d_pair(b, mb, full, kb * 64, n0, pl, keep);
            }
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // -------------------------------------------------------------- MMA issuer (leader only)
    if (rank == 0 && ptx::elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true;
      for (int tile = pair_id; tile < num_tiles && ok; tile += num_pairs) {
        int m0, n0;
        const Product &p = prob.p[decode(tile, m0, n0)];
        const bool a_mn = p.a_mn != 0, b_mn = p.b_mn != 0;
        const uint32_t idesc = ptx::make_idesc(1u, std::is_same<T, __half>::value ? 0u : 1u, kPairTileM, BN) |
                               (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
        // leading byte offset of an MN-major operand; 16 of K are 16 rows there, 32 bytes of a row otherwise
        const uint64_t a_lbo = a_mn ? (uint64_t)(kChunkBytes >> 4) << 16 : 0, b_lbo = b_mn ? (uint64_t)(kChunkBytes >> 4) << 16 : 0;
        const uint32_t a_step = a_mn ? (16 * kRowBytes) >> 4 : 2, b_step = b_mn ? (16 * kRowBytes) >> 4 : 2;
        for (int kb0 = 0; kb0 < p.kblocks && ok; kb0 += prob.chunk, ++local) {
          const int buf = local & 1;
          if (!ptx::mbar_wait(tmem_empty + buf, ((uint32_t)(local >> 1) & 1u) ^ 1u, abort_flag)) {
            gave_up(kStatusMmaTimeout);
            ok = false;
            break;
          }
          ptx::tc_fence_after_sync();
          const uint32_t d = tmem_base + (uint32_t)(buf * BN);
          uint32_t accumulate = 0;
          const int kb1 = kb0 + prob.chunk < p.kblocks ? kb0 + prob.chunk : p.kblocks;
          for (int kb = kb0; kb < kb1; ++kb) {
            if (!ptx::mbar_wait(full_bar + stage, phase, abort_flag)) {
              gave_up(kStatusMmaTimeout);
              ok = false;
              break;
            }
            ptx::tc_fence_after_sync();
            const uint32_t st = ptx::smem_u32(smem + stage * kStageBytes);
            // pieces whose product is below fp32 resolution of the leading one (pa + pb > 2) are skipped; the small ones
            // come first, while the accumulator is small and its truncation with it
#pragma unroll
            for (int sum = PL - 1; sum >= 0; --sum)
#pragma unroll
              for (int pa = 0; pa <= sum; ++pa) {
                const uint64_t ad = ptx::smem_desc_k_sw128(st + pa * kABytes) | a_lbo;
                const uint64_t bd = ptx::smem_desc_k_sw128(st + PL * kABytes + (sum - pa) * kBBytes) | b_lbo;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  ptx::mma_pair_bf16(d, ad + k * a_step, bd + k * b_step, idesc, accumulate);
                  accumulate = 1;
                }
              }
            ptx::mma_commit_pair(ptx::smem_u32(empty_bar + stage)); // frees the stage in both CTAs
            ptx::mma_commit_pair(ptx::map_to_cta(ptx::smem_u32(empty_bar + stage), 1));
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (ok) {
            ptx::mma_commit_pair(ptx::smem_u32(tmem_full + buf));
            ptx::mma_commit_pair(ptx::map_to_cta(ptx::smem_u32(tmem_full + buf), 1));
          }
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- epilogue (both CTAs): a thread a row
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lanes = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const LossRows &rows = prob.rows;
    float *stg = stage_out + (warp - 2) * (32 * 33);
    int local = 0;
    bool ok = true;
    float acc[2 * kMyChunks][16]; // 16 columns at a time: with 32 the sums and a chunk do not fit in 168 registers
    for (int tile = pair_id; tile < num_tiles && ok; tile += num_pairs) {
      int m0, n0;
      const Product &p = prob.p[decode(tile, m0, n0)];
      const int row_base = m0 + (int)rank * kTileM + quarter * 32, row = row_base + lane;
      const bool row_ok = row < p.M;
      int64_t label = -1;
      float top = 0.0f, log2_sum = 0.0f, factor = 0.0f, undo = 1.0f;
      if constexpr (kOut == Out::kStore) {
        undo = rows.scale[2];
      } else {
        if (row_ok) {
          label = rows.label_of(row);
          if constexpr (kOut == Out::kGrad) {
            const float2 s = rows.stat[row];
            top = s.x, log2_sum = s.y * kLog2e;
            factor = label < 0 ? 0.0f : label >= rows.classes ? NAN : __fdiv_rn(rows.dloss[row], rows.scale[0]) * rows.scale[1];
          }
        }
      }
      // K in chunks: all but the last go to registers
      const int chunks = (p.kblocks + prob.chunk - 1) / prob.chunk;
      MaxSum t{-INFINITY, 0.0f};
      for (int kc = 0; kc < chunks && ok; ++kc, ++local) {
        const int buf = local & 1;
        const bool got = ptx::mbar_wait(tmem_full + buf, (uint32_t)(local >> 1) & 1u, abort_flag);
        if (!__all_sync(0xffffffffu, got)) {
          if (lane == 0)
            gave_up(kStatusEpilogueTimeout);
          ok = false;
          break;
        }
        ptx::tc_fence_after_sync();
        const bool last = kc + 1 == chunks;
#pragma unroll
        for (int ci = 0; ci < kMyChunks; ++ci) {
          const int c0 = 32 * half + 64 * ci, col0 = n0 + c0;
          if (col0 >= p.N)
            break;
          if (kOut != Out::kSums)
            __syncwarp(); // (the staged chunk before has been read)
          const int64_t mine = label - prob.class0 - col0; // the label's column in this chunk, if in [0, 32)
          float b_lane = 0.0f;
          if constexpr (kOut != Out::kStore)
            if (prob.bias && last && col0 + lane < p.N)
              b_lane = to_f32(static_cast<const T *>(prob.bias)[prob.class0 + col0 + lane]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t r[16];
            float(&sum)[16] = acc[2 * ci + h];
            ptx::tmem_ld_32x16(lanes + (uint32_t)(buf * BN + c0 + 16 * h), r);
            ptx::tmem_ld_wait();
            if (row_base >= p.M)
              continue;
            if (!last) {
#pragma unroll
              for (int j = 0; j < 16; ++j)
                sum[j] = kc == 0 ? __uint_as_float(r[j]) : __fadd_rn(sum[j], __uint_as_float(r[j]));
              continue;
            }
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j)
              v[j] = kc == 0 ? __uint_as_float(r[j]) : __fadd_rn(sum[j], __uint_as_float(r[j]));
            if constexpr (kOut == Out::kStore) {
#pragma unroll
              for (int j = 0; j < 16; ++j)
                v[j] *= undo;
            } else {
              if (prob.bias)
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  v[j] += __shfl_sync(0xffffffffu, b_lane, 16 * h + j);
              const int here = mine >= 16 * h && mine < 16 * h + 16 ? (int)mine - 16 * h : -1;
              if constexpr (kOut == Out::kSums) {
                if (col0 + 16 * h + 16 > p.N)
#pragma unroll
                  for (int j = 0; j < 16; ++j)
                    if (col0 + 16 * h + j >= p.N)
                      v[j] = -INFINITY;
                if (here >= 0) {
                  float l = 0.0f;
#pragma unroll
                  for (int j = 0; j < 16; ++j)
                    l = j == here ? v[j] : l;
                  rows.target[row] = l;
                }
                float m = t.m;
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  m = fmaxf(m, v[j]);
                const float b = m == -INFINITY ? 0.0f : m;
                float s = t.s * ex2((t.m - b) * kLog2e);
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  s += ex2((v[j] - b) * kLog2e);
                t = {m, s};
              } else {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  v[j] = ex2(fmaf(v[j] - top, kLog2e, -log2_sum));
                if (here >= 0)
#pragma unroll
                  for (int j = 0; j < 16; ++j)
                    v[j] -= j == here ? 1.0f : 0.0f;
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  v[j] = label < 0 ? 0.0f : v[j] * factor;
              }
            }
            if constexpr (kOut != Out::kSums)
#pragma unroll
              for (int j = 0; j < 16; ++j)
                stg[lane * 33 + 16 * h + j] = v[j];
          }
          if (row_base >= p.M || !last)
            continue;
          if constexpr (kOut != Out::kSums) {
            __syncwarp();
            const int rows_here = p.M - row_base < 32 ? p.M - row_base : 32, cols_here = p.N - col0 < 32 ? p.N - col0 : 32;
            if constexpr (kOut == Out::kGrad && kF32) {
              __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out) + (int64_t)row_base * p.ldo + col0;
#pragma unroll 4
              for (int i = 0; i < rows_here; ++i) {
                float f = stg[i * 33 + lane];
                if (lane < cols_here)
#pragma unroll
                  for (int pl = 0; pl < 3; ++pl) {
                    const __nv_bfloat16 h = __float2bfloat16_rn(f);
                    out[pl * p.plane + i * p.ldo + lane] = h;
                    f = __fsub_rn(f, __bfloat162float(h));
                  }
              }
            } else if (kF32 || p.out_f32) {
              float *out = static_cast<float *>(p.out) + (int64_t)row_base * p.ldo + col0 + lane;
              const float *base = p.base ? p.base + (int64_t)row_base * p.ldo + col0 + lane : nullptr;
#pragma unroll 8
              for (int i = 0; i < rows_here; ++i) {
                if (lane >= cols_here)
                  continue;
                float f = stg[i * 33 + lane];
                if (base)
                  f += base[i * p.ldo];
                if (p.accum)
                  f += out[i * p.ldo];
                out[i * p.ldo] = f;
              }
            } else if constexpr (!kF32) {
              // two columns a lane, two rows an instruction, where the pairs are aligned
              T *out = static_cast<T *>(p.out) + (int64_t)row_base * p.ldo + col0;
              const float *base = p.base ? p.base + (int64_t)row_base * p.ldo + col0 : nullptr;
              if (cols_here == 32 && (p.ldo & 1) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 3) == 0) {
                const int c = 2 * (lane & 15);
#pragma unroll 8
                for (int i = lane >> 4; i < rows_here; i += 2) {
                  float f[2] = {stg[i * 33 + c], stg[i * 33 + c + 1]};
                  if (base)
                    f[0] += base[i * p.ldo + c], f[1] += base[i * p.ldo + c + 1];
                  if (p.accum) {
                    const Pack<T, 2> old = load_pack<T, 2>(out + i * p.ldo + c);
                    f[0] += old.f(0), f[1] += old.f(1);
                  }
                  store_pack<T, 2>(out + i * p.ldo + c, f);
                }
              } else {
#pragma unroll 4
                for (int i = 0; i < rows_here; ++i) {
                  if (lane >= cols_here)
                    continue;
                  float f = stg[i * 33 + lane];
                  if (base)
                    f += base[i * p.ldo + lane];
                  if (p.accum)
                    f += to_f32(out[i * p.ldo + lane]);
                  out[i * p.ldo + lane] = from_f32<T>(f);
                }
              }
            }
          }
        }
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0)
          ptx::mbar_arrive_cluster(ptx::map_to_cta(ptx::smem_u32(tmem_empty + buf), 0));
      }
      if constexpr (kOut == Out::kSums)
        if (ok && row_ok)
          rows.partial[(int64_t)row * rows.tiles + n0 / BN * 2 + half] = make_float2(t.m, t.s);
    }
  }

  // ------------------------------------------------------------------ teardown
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag != 0) { // copies in flight land before the shared memory is given up
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 2000000ull)
      __nanosleep(1000);
    __syncthreads();
  }
  ptx::cluster_sync(); // neither CTA leaves while its peer may still signal its barriers
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

// An operand in memory: [planes][rows][pitch] of 16-bit values, 16-byte aligned, pitch a multiple of 8.
struct Operand {
  const void *p;
  int64_t rows, cols, pitch, plane_rows;
  int planes;
  const void *at(int64_t col) const { return static_cast<const char *>(p) + 2 * col; }
};
inline int loss_operand_map(CUtensorMap *map, const Operand &o, bool mn, int box_rows) {
  const uint64_t dims[3] = {(uint64_t)o.cols, (uint64_t)o.rows, (uint64_t)o.planes};
  const uint64_t strides[2] = {(uint64_t)o.pitch * 2, (uint64_t)(o.pitch * o.plane_rows) * 2};
  const uint32_t box[3] = {64, mn ? 64u : (uint32_t)box_rows, 1};
  return encode_tiled(map, 0, 3, o.p, dims, strides, box, nullptr, 128);
}

// The launch of up to two products: operands a[i] (M side) and b[i] (N side).
template <typename T, int BN, Out kOut>
inline int launch_loss_gemm(const Products &in, const Operand *a, const Operand *b, cudaStream_t st) {
  constexpr int PL = std::is_same<T, float>::value ? 3 : 1;
  auto kernel = loss_gemm_kernel<T, BN, kOut>;
  constexpr size_t smem = loss_smem_bytes<PL, BN>();
  static_assert(smem <= 227 * 1024, "shared memory budget");
  static std::atomic<bool> configured[64]{};
  int dev = 0;
  NB_CUDA(cudaGetDevice(&dev));
  if (!configured[dev & 63]) {
    NB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    configured[dev & 63] = true;
  }
  Products prob = in;
  // 16 bits: 96 steps (an error of 1.4e-6 of the result's RMS, and three times that after a thousand); fp32: a K block, whose
  // last four steps are the only ones on a large accumulator
  prob.chunk = PL == 3 ? 1 : 24;
  CUtensorMap ma[2], mb[2];
  int tiles = 0;
  for (int i = 0; i < prob.count; ++i) {
    Product &p = prob.p[i];
    p.m_tiles = (p.M + kPairTileM - 1) / kPairTileM;
    p.n_tiles = (p.N + BN - 1) / BN;
    tiles += p.m_tiles * p.n_tiles;
    NB_TRY(loss_operand_map(&ma[i], a[i], p.a_mn, kTileM));
    NB_TRY(loss_operand_map(&mb[i], b[i], p.b_mn, BN / 2));
  }
  if (prob.count == 1)
    ma[1] = ma[0], mb[1] = mb[0];
  int *status = nullptr;
  NB_TRY(device_status_word(&status));
  const int pairs = std::min(sm_count() / 2, tiles);
  NB_CUDA(launch_dependent(kernel, dim3(2 * pairs), dim3(kPairThreads), smem, st, ma[0], mb[0], ma[1], mb[1], prob, status));
  return NB200_OK;
}

} // namespace nb200
