// The products of a classifying head on tcgen05: l = x W, dx = G W^T, dW = x^T G, each from the operands as they lie.
//
// W [inputs, classes] has its classes in neighbouring memory, so in l = x W, and for both operands of dW, the rows of memory
// run along K: those operands are read as MN-major ones, stored as chunks of 64 rows (K) x 128 bytes (bit 15 / 16 of the
// instruction descriptor; the leading byte offset leads from one chunk of 64 columns to the next). Nothing is transposed.
//
// Two shapes (kPair): clusters of two CTAs that make 256 x 256 tiles (cta_group::2: each loads its own 128 rows of A and 128
// columns of B by TMA, the leader issues the MMAs, both drain their 128 accumulator rows), and single CTAs with 128 x 64 tiles
// for products whose large tiles would leave most SMs idle.
//
// PL planes an operand: 1 (bf16 or fp16 as it is) or 3 (the bf16 pieces of an fp32 tensor; the six products that matter at
// fp32 resolution). The tensor core's additions truncate: every few MMA steps the accumulator is added up in fp32 registers
// (gemm.cuh).
//
// What becomes of a tile, by the epilogue, in which a thread owns a row:
//   kSums   of each row and half of a tile's column chunks, the maximum and the sum of the exponentials; the label's logit
//   kGrad   G, in 16 bits (fp32: three bf16 planes)
//   kStore  the product itself, two products (dx and dW of a piece of the classes) in one launch: with one after the other,
//           each would end in a round of tiles that leaves SMs idle
//
// Bound by the tensor pipe: 1400 to 1600 TFLOP/s in bf16 ([8192, 2048] . [2048, 128000]: the logits 2.68 ms, G of a piece of 4096
// classes 98 us, both gradients of such a piece 193), which the power limit brings down to 1240 over a whole step.
#pragma once
#include "gemm2.cuh"
#include "loss_plan.h"
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
  int M, N, K, kblocks, m_tiles, n_tiles;
  int steps;    // MMA steps of a K block: four, or what a single short block needs
  int tx_bytes; // that a stage's loads bring to a CTA
  int splits, split_blocks; // kStore: K in `splits` tiles of split_blocks K blocks, each with a result of its own
  int a_mn, b_mn;           // memory rows run along K
  // kStore: out [splits][M][ldo] (+)= scale[2] * D; kGrad: out is G [planes][M][ldo]. stride: between splits or planes
  void *out;
  int64_t ldo, stride;
  int out_f32, accum;
  int vec; // rows of out begin at 16-byte boundaries
  // kSplit: B in memory, b_rows x b_cols fp32 values at a pitch of b_ld; rows begin at 8-byte boundaries
  const float *b;
  int64_t b_rows, b_cols, b_ld;
  int b_pairs;
};
struct Products {
  Product p[kMaxProducts];
  int count;
  int extra_tiles; // see the kernel's tile_at
  int chunk;  // K blocks accumulated in tensor memory
  int class0; // kSums, kGrad: the class of the first column
  const void *bias;
  LossRows rows;
};

// kLong: K goes through tensor memory in more than one chunk, and the chunks' sums take an epilogue thread 128 registers; eight
// epilogue warps. Without them there is room for sixteen (16 bits; three planes leave no shared memory for their buffers), which
// a short K needs: its tiles are bound by the epilogue's latencies (K = 302: 1900 cycles a 16-column step with two warps a
// scheduler, 2560 cycles of MMAs a tile of 256 columns). What the sums make the compiler spill costs more than its bytes: beside
// so much shared memory the L1 keeps none of it (fp32 dW of 32 rows, [2048, 65536]: 246 us with them, 132 without, and with rows
// of 128 bytes a store).
// kSplit (fp32, one CTA, 128 x 128 tiles): eight more warps make the pieces of B from the fp32 values on their way to shared
// memory. Bound by its bandwidth: of some 2600 cycles a K block 2300 are the 192 KB that its 24 MMAs read, 48 KB of W's pieces and
// 48 of x's ([32, 2048] . [2048, 65536] 197 us, bytes 82; [32, 2048] . [2048, 100000] 275 us, 400 with four such warps).
template <int PL, bool kPair, bool kLong, bool kSplit> struct LossShape {
  static_assert(!kSplit || (PL == 3 && !kPair && kLong), "only fp32 has pieces");
  static constexpr int kWarps = kPair && !kLong && PL == 1 ? 16 : 8; // of the epilogue
  static constexpr int kSplitters = kSplit ? 8 : 0;                  // warps that make pieces
  static constexpr int kThreads = 32 * (2 + kWarps + kSplitters);
  static constexpr int kTileRows = kPair ? 256 : 128, kTileCols = kPair ? 256 : kSplit ? 128 : 64; // of a cluster
  static constexpr int kCtaCols = kPair || kSplit ? 128 : 64;                                      // columns of B that a CTA loads
  static constexpr uint32_t kABytes = kTileM * kRowBytes, kBBytes = kCtaCols * kRowBytes;
  static constexpr uint32_t kStageBytes = PL * (kABytes + kBBytes);
  static constexpr int kStages = PL == 3 ? 2 : kWarps == 16 ? 5 : 6;
  static constexpr int kPitch = PL == 3 ? 33 : 32;   // of an epilogue warp's transpose buffer; 33: offsets that are constants
  static constexpr int kWarpStage = 32 * kPitch * 4; // its bytes
  static constexpr size_t kSmem =
      (size_t)kStages * kStageBytes + kWarps * kWarpStage + (2 * kStages + 4) * 8 + 16 + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory budget");
};

__device__ __forceinline__ void add_f32x4(float *p, const float *v) { // (one writer an element and launch: no order to vary)
  asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
}
template <typename T> __device__ __forceinline__ void store16(T *p, const float (&v)[16]) {
  constexpr int V = kPackOf<T>;
#pragma unroll
  for (int q = 0; q < 16 / V; ++q) {
    float o[V];
#pragma unroll
    for (int j = 0; j < V; ++j)
      o[j] = v[q * V + j];
    store_pack<T, V>(p + q * V, o);
  }
}

// T: the operands' type; float means three bf16 planes.
template <typename T, bool kPair, bool kLong, Out kOut, bool kSplit>
__global__ void __launch_bounds__(LossShape<std::is_same<T, float>::value ? 3 : 1, kPair, kLong, kSplit>::kThreads, 1)
    loss_gemm_kernel(const __grid_constant__ CUtensorMap map_a0, const __grid_constant__ CUtensorMap map_b0,
                     const __grid_constant__ CUtensorMap map_a1, const __grid_constant__ CUtensorMap map_b1,
                     const __grid_constant__ Products prob, int *status) {
  constexpr bool kF32 = std::is_same<T, float>::value;
  constexpr int PL = kF32 ? 3 : 1;
  using S = LossShape<PL, kPair, kLong, kSplit>;
  constexpr int STAGES = S::kStages, BN = S::kTileCols;
  constexpr uint32_t kABytes = S::kABytes, kBBytes = S::kBBytes, kStageBytes = S::kStageBytes;
  constexpr uint32_t kChunkBytes = 64 * kRowBytes; // 64 columns x 64 of K of an MN-major operand
  constexpr int kParts = S::kWarps / 4;            // epilogue warps that share the rows of a quarter
  constexpr int kMyChunks = BN / (32 * kParts);    // column chunks of 32 that each drains
  constexpr uint32_t kTmemCols = 2 * BN;
  constexpr uint32_t kCtas = kPair ? 2 : 1;

  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float *stage_out = reinterpret_cast<float *>(smem + STAGES * kStageBytes);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + STAGES * kStageBytes + S::kWarps * S::kWarpStage);
  uint64_t *full_bar = bars, *empty_bar = bars + STAGES, *tmem_full = bars + 2 * STAGES, *tmem_empty = tmem_full + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tmem_empty + 2);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = kPair ? ptx::cluster_ctarank() : 0; // 0 = leader
  const int unit = kPair ? blockIdx.x >> 1 : blockIdx.x, units = kPair ? gridDim.x >> 1 : gridDim.x;
  const int tiles0 = prob.p[0].m_tiles * prob.p[0].n_tiles * prob.p[0].splits;
  const int num_tiles =
      tiles0 + (kOut == Out::kStore && prob.count > 1 ? prob.p[1].m_tiles * prob.p[1].n_tiles * prob.p[1].splits : 0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      ptx::mbar_init(full_bar + s, 1 + S::kSplitters);
      ptx::mbar_init(empty_bar + s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      ptx::mbar_init(tmem_full + b, 1);
      ptx::mbar_init(tmem_empty + b, kCtas * S::kWarps);
    }
    *abort_flag = 0;
    ptx::mbar_fence_init();
    ptx::prefetch_tensormap(&map_a0);
    ptx::prefetch_tensormap(&map_b0);
  }
  if (warp == 1) {
    if (kPair) {
      ptx::tmem_alloc_pair(tmem_slot, kTmemCols);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(tmem_slot, kTmemCols);
      ptx::tmem_relinquish();
    }
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (kPair)
    ptx::cluster_sync(); // the peer's barriers are initialised before anything is signalled remotely
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  if (num_tiles <= units) // one round of tiles (early_trigger's reason)
    pdl_trigger();

  auto gave_up = [&](int code) {
    if (*abort_flag == 0)
      atomicCAS(status, 0, code);
    *abort_flag = 1;
  };
  // A tile's product, first row and column, split and K blocks [kb0, kb1). Rows vary fastest, so that the tiles in flight
  // share columns of B (a short K: columns).
  struct At {
    int which, m0, n0, split, kb0, kb1;
  };
  auto decode = [&](int tile) {
    At t;
    t.which = kOut == Out::kStore && tile >= tiles0 ? 1 : 0;
    const Product &p = prob.p[t.which];
    tile -= t.which ? tiles0 : 0;
    if (kOut == Out::kStore && p.splits == 1 && p.kblocks <= 2) { // its stores bound it: runs of neighbouring columns
      t.n0 = tile % p.n_tiles * BN;
      t.m0 = tile / p.n_tiles * S::kTileRows;
      t.split = 0;
    } else {
      t.m0 = tile % p.m_tiles * S::kTileRows;
      tile /= p.m_tiles;
      t.n0 = tile % p.n_tiles * BN;
      t.split = tile / p.n_tiles;
    }
    t.kb0 = t.split * p.split_blocks;
    t.kb1 = t.kb0 + p.split_blocks < p.kblocks ? t.kb0 + p.split_blocks : p.kblocks;
    return t;
  };
  // This unit's i-th tile, or -1: the first product's dealt out one by one; of the second's, `extra_tiles` to each of the units
  // that got one more of the first, the rest to the others.
  const int more = tiles0 % units, own0 = tiles0 / units + (unit < more ? 1 : 0);
  auto tile_at = [&](int i) -> int {
    if (i < own0)
      return unit + i * units;
    if (kOut != Out::kStore || num_tiles == tiles0)
      return -1;
    i -= own0;
    int t;
    if (unit < more)
      t = i < prob.extra_tiles ? unit + i * more : num_tiles;
    else
      t = more * prob.extra_tiles + (unit - more) + i * (units - more);
    return t < num_tiles - tiles0 ? tiles0 + t : -1;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (every CTA)
    if (ptx::elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint64_t keep = ptx::l2_policy_evict_last();
      for (int i = 0, tile; ok && (tile = tile_at(i)) >= 0; ++i) {
        const At t = decode(tile);
        const bool a_mn = prob.p[t.which].a_mn != 0, b_mn = prob.p[t.which].b_mn != 0;
        const CUtensorMap *ma = t.which ? &map_a1 : &map_a0, *mb = t.which ? &map_b1 : &map_b0;
        const int m0 = t.m0 + (int)rank * kTileM, n0 = t.n0 + (int)rank * S::kCtaCols;
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          if (!ptx::mbar_wait(empty_bar + stage, phase ^ 1u, abort_flag)) {
            gave_up(kStatusProducerTimeout);
            ok = false;
            break;
          }
          uint8_t *st = smem + stage * kStageBytes;
          const uint32_t full = kPair ? ptx::map_to_cta(ptx::smem_u32(full_bar + stage), 0) : 0;
          if (rank == 0)
            ptx::mbar_expect_tx(full_bar + stage, kCtas * (uint32_t)prob.p[t.which].tx_bytes); // bytes of both CTAs
          auto load = [&](uint8_t *dst, const CUtensorMap *map, int c0, int c1, int pl) {
            if constexpr (kPair)
              ptx::tma_load_3d_pair(dst, map, full, c0, c1, pl, keep);
            else
              ptx::tma_load_3d(dst, map, full_bar + stage, c0, c1, pl);
          };
#pragma unroll
          for (int pl = 0; pl < PL; ++pl) {
            uint8_t *a = st + pl * kABytes, *b = st + PL * kABytes + pl * kBBytes;
            if (a_mn) {
#pragma unroll
              for (int j = 0; j < kTileM / 64; ++j)
                load(a + j * kChunkBytes, ma, m0 + 64 * j, kb * 64, pl);
            } else {
              load(a, ma, kb * 64, m0, pl);
            }
            if constexpr (kSplit)
              continue;
            if (b_mn) {
#pragma unroll
              for (int j = 0; j < S::kCtaCols / 64; ++j)
                load(b + j * kChunkBytes, mb, n0 + 64 * j, kb * 64, pl);
            } else {
              load(b, mb, kb * 64, n0, pl);
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
      auto commit = [&](uint64_t *bar) { // on every CTA's barrier, when the MMAs so far have finished
        if constexpr (kPair) {
          ptx::mma_commit_pair(ptx::smem_u32(bar));
          ptx::mma_commit_pair(ptx::map_to_cta(ptx::smem_u32(bar), 1));
        } else {
          ptx::mma_commit(bar);
        }
      };
      for (int i = 0, tile; ok && (tile = tile_at(i)) >= 0; ++i) {
        const At t = decode(tile);
        const bool a_mn = prob.p[t.which].a_mn != 0, b_mn = prob.p[t.which].b_mn != 0;
        const uint32_t idesc = ptx::make_idesc(1u, std::is_same<T, __half>::value ? 0u : 1u, S::kTileRows, BN) |
                               (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
        // leading byte offset of an MN-major operand; 16 of K are 16 rows there, 32 bytes of a row otherwise
        const uint64_t a_lbo = a_mn ? (uint64_t)(kChunkBytes >> 4) << 16 : 0, b_lbo = b_mn ? (uint64_t)(kChunkBytes >> 4) << 16 : 0;
        const int steps = prob.p[t.which].steps;
        const uint32_t a_step = a_mn ? (16 * kRowBytes) >> 4 : 2, b_step = b_mn ? (16 * kRowBytes) >> 4 : 2;
        for (int kb0 = t.kb0; kb0 < t.kb1 && ok; kb0 += prob.chunk, ++local) {
          const int buf = local & 1;
          if (!ptx::mbar_wait(tmem_empty + buf, ((uint32_t)(local >> 1) & 1u) ^ 1u, abort_flag)) {
            gave_up(kStatusMmaTimeout);
            ok = false;
            break;
          }
          ptx::tc_fence_after_sync();
          const uint32_t d = tmem_base + (uint32_t)(buf * BN);
          uint32_t accumulate = 0;
          const int kb1 = kb0 + prob.chunk < t.kb1 ? kb0 + prob.chunk : t.kb1;
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
                  if (k >= steps)
                    break;
                  if constexpr (kPair)
                    ptx::mma_pair_bf16(d, ad + k * a_step, bd + k * b_step, idesc, accumulate);
                  else
                    ptx::mma_bf16(d, ad + k * a_step, bd + k * b_step, idesc, accumulate);
                  accumulate = 1;
                }
              }
            commit(empty_bar + stage); // frees the stage
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (ok)
            commit(tmem_full + buf);
        }
      }
    }
  } else if (kSplit && warp >= 2 + S::kWarps) {
    // ---------------------------------------------------------------- pieces of B
    // A K block of B is 128 runs of 64 neighbouring fp32 values: run u is a row of W, its pieces 128 bytes of shared memory each.
    // This warp has the runs me, me + 8, ..., a lane two values of each; the next block's are on their way to registers while one
    // is multiplied, the one behind it to L2 (4096 x 131071 fp32 3 % less time).
    if constexpr (kSplit) {
      constexpr int kApart = S::kSplitters, kRuns = 128 / kApart;
      constexpr bool kMn = kOut != Out::kStore; // the runs of a K block: 64 of K for each of two groups of columns, or 128 columns
      const int me = warp - (2 + S::kWarps);
      const Product &p = prob.p[0];
      static_assert(kApart == 8, "a run's number in eight is the warp's");
      const uint32_t at = (uint32_t)me * kRowBytes + ((lane >> 2) ^ me) * 16 + (lane & 3) * 4; // (128-byte swizzle)
      const int64_t step = kApart * p.b_ld;
      int next_i = 0, next_kb = 0;
      bool more = true;
      At next{};
      const float *from = nullptr; // of the next block: this lane's values of the warp's first run
      int x_rows[2], y_rows[2];    // its rows that hold this lane's first value, and its second, of each group of columns
      auto seek = [&]() {
        const int64_t row = (kMn ? next_kb * 64 : next.n0) + me, col = (kMn ? next.n0 : next_kb * 64) + 2 * lane;
        from = p.b + row * p.b_ld + col;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const int rows_left = more ? (int)(p.b_rows - row) : 0, cols_left = (int)(p.b_cols - col) - 64 * g;
          x_rows[g] = cols_left > 0 ? rows_left : 0, y_rows[g] = cols_left > 1 ? rows_left : 0;
        }
        // the block behind it on its way to L2: a lane half a run
        const int run = lane & 15, half = lane >> 4;
        const int64_t r = row + kApart * (kMn ? run & 7 : run) + (kMn ? 64 : 0);
        const int64_t c = col - 2 * lane + (kMn ? 64 * (run >> 3) : 64) + 32 * half;
        if (more && next_kb + 1 < next.kb1 && r < p.b_rows && c < p.b_cols)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(p.b + r * p.b_ld + c));
      };
      auto first_of_tile = [&]() {
        const int tile = tile_at(next_i);
        more = tile >= 0;
        if (more)
          next = decode(tile), next_kb = next.kb0;
        seek();
      };
      auto make = [&](auto pairs) { // pairs: rows begin at 8-byte boundaries, and have an even number of values
        float2 v[kRuns];
        const float *q = from;
        auto fetch = [&](int i) {
          const int g = kMn ? i / (kRuns / 2) : 0, row = kApart * (kMn ? i % (kRuns / 2) : i);
          if (kMn && i == kRuns / 2)
            q = from + 64;
          v[i] = make_float2(0.0f, 0.0f);
          if constexpr (decltype(pairs)::value) {
            if (row < y_rows[g])
              v[i] = *reinterpret_cast<const float2 *>(q);
          } else {
            if (row < x_rows[g])
              v[i].x = q[0];
            if (row < y_rows[g])
              v[i].y = q[1];
          }
          q += step;
        };
#pragma unroll
        for (int i = 0; i < kRuns; ++i)
          fetch(i);
        int stage = 0;
        uint32_t phase = 0;
        while (more) {
          if (!__all_sync(0xffffffffu, ptx::mbar_wait(empty_bar + stage, phase ^ 1u, abort_flag))) {
            if (lane == 0)
              gave_up(kStatusProducerTimeout);
            break;
          }
          if (++next_kb < next.kb1)
            seek();
          else
            ++next_i, first_of_tile();
          q = from;
          uint8_t *b = smem + stage * kStageBytes + PL * kABytes + at;
#pragma unroll
          for (int i = 0; i < kRuns; ++i) {
            float2 left = v[i];
#pragma unroll
            for (int pl = 0; pl < PL; ++pl) {
              const __nv_bfloat162 h = __floats2bfloat162_rn(left.x, left.y);
              const uint32_t bits = *reinterpret_cast<const uint32_t *>(&h);
              *reinterpret_cast<uint32_t *>(b + pl * kBBytes + i * (kApart * kRowBytes)) = bits;
              left.x = __fsub_rn(left.x, __uint_as_float(bits << 16));
              left.y = __fsub_rn(left.y, __uint_as_float(bits & 0xffff0000u));
            }
          }
          ptx::fence_async_shared();
          __syncwarp();
          if (lane == 0)
            ptx::mbar_arrive(full_bar + stage);
#pragma unroll
          for (int i = 0; i < kRuns; ++i)
            fetch(i);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      };
      first_of_tile();
      if (p.b_pairs)
        make(std::true_type{});
      else
        make(std::false_type{});
    }
  } else {
    // ---------------------------------------------------------------- epilogue (every CTA): a thread a row
    const int quarter = warp & 3, part = (warp - 2) >> 2;
    const uint32_t lanes = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const LossRows &rows = prob.rows;
    float *stg = stage_out + (warp - 2) * (S::kWarpStage / 4);
    int local = 0;
    bool ok = true;
    float acc[kLong ? 2 * kMyChunks : 1][16]; // 16 columns at a time: with 32 the sums and a chunk do not fit in 168 registers
    for (int i = 0, tile; ok && (tile = tile_at(i)) >= 0; ++i) {
      const At at = decode(tile);
      const Product &p = prob.p[at.which];
      const int M = p.M, N = p.N, n0 = at.n0;
      const int row_base = at.m0 + (int)rank * kTileM + quarter * 32, row = row_base + lane;
      const bool row_ok = row < M;
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
      // kStore: this thread's row of the result, and whether its 16-byte accesses are aligned
      const int64_t ldo = p.ldo;
      const bool vec = p.vec != 0, accum = p.accum != 0, out_f32 = kF32 || p.out_f32 != 0;
      const bool staged = kOut == Out::kStore && !kLong && vec && out_f32 && !accum;
      const int64_t out0 = at.split * p.stride;
      const int chunks = (at.kb1 - at.kb0 + prob.chunk - 1) / prob.chunk;
      MaxSum t{-INFINITY, 0.0f};
      if constexpr (kOut != Out::kStore)
        if (prob.bias) { // this warp's columns of it, while the tile is being made
          __syncwarp();
#pragma unroll
          for (int ci = 0; ci < kMyChunks; ++ci) {
            const int c = n0 + 32 * part + 32 * kParts * ci + lane;
            stg[32 * ci + lane] = c < N ? to_f32(static_cast<const T *>(prob.bias)[prob.class0 + c]) : 0.0f;
          }
          __syncwarp();
        }
      // What becomes of 16 columns of this thread's row, v: the h-th half of the warp's ci-th chunk of 32.
      auto finish = [&](int ci, int h, float(&v)[16]) {
        const int col0 = n0 + 32 * part + 32 * kParts * ci;
        const int mine = (int)(label - prob.class0 - col0); // the label's column in this chunk, if in [0, 32)
        const int col = col0 + 16 * h;
        if constexpr (kOut == Out::kStore) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            v[j] *= undo;
          if (!vec) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              stg[lane * S::kPitch + (kF32 ? 16 * h + j : (16 * h + j) ^ lane)] = v[j];
          } else if (staged) {
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              *reinterpret_cast<float4 *>(stg + lane * 32 + ((16 * h + j) ^ (lane & 7) * 4)) =
                  make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          } else if (row_ok && col < N) {
            const int64_t off = out0 + (int64_t)row * ldo + col;
            if (out_f32) {
              float *out = static_cast<float *>(p.out) + off;
              if (col + 16 > N) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  if (col + j < N)
                    out[j] = accum ? out[j] + v[j] : v[j];
              } else if (accum) {
#pragma unroll
                for (int j = 0; j < 16; j += 4)
                  add_f32x4(out + j, v + j);
              } else {
                store16<float>(out, v);
              }
            } else if constexpr (!kF32) {
              T *out = static_cast<T *>(p.out) + off;
              if (col + 16 > N) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  if (col + j < N)
                    out[j] = from_f32<T>(accum ? to_f32(out[j]) + v[j] : v[j]);
              } else {
                if (accum) {
                  const Pack<T, 8> o0 = load_pack<T, 8>(out), o1 = load_pack<T, 8>(out + 8);
#pragma unroll
                  for (int j = 0; j < 8; ++j)
                    v[j] += o0.f(j), v[8 + j] += o1.f(j);
                }
                store16<T>(out, v);
              }
            }
          }
        } else {
          if (prob.bias)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
              const float4 b = *reinterpret_cast<const float4 *>(stg + 32 * ci + 16 * h + j);
              v[j] += b.x, v[j + 1] += b.y, v[j + 2] += b.z, v[j + 3] += b.w;
            }
          const int here = mine >= 16 * h && mine < 16 * h + 16 ? mine - 16 * h : -1;
          if constexpr (kOut == Out::kSums) {
            if (col + 16 > N)
#pragma unroll
              for (int j = 0; j < 16; ++j)
                if (col + j >= N)
                  v[j] = -INFINITY;
            if (here >= 0) {
              float l = 0.0f;
#pragma unroll
              for (int j = 0; j < 16; ++j)
                l = j == here ? v[j] : l;
              rows.target[row] = l;
            }
            float m4[4] = {t.m, v[1], v[2], v[3]}; // four chains each, for their latency
            m4[0] = fmaxf(m4[0], v[0]);
#pragma unroll
            for (int j = 4; j < 16; ++j)
              m4[j & 3] = fmaxf(m4[j & 3], v[j]);
            const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
            const float b = m == -INFINITY ? 0.0f : m;
            float s4[4] = {t.s * ex2((t.m - b) * kLog2e), 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < 16; ++j)
              s4[j & 3] += ex2((v[j] - b) * kLog2e);
            t = {m, (s4[0] + s4[1]) + (s4[2] + s4[3])};
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
            if (row_ok) { // (G's rows are as wide as whole tiles)
              if constexpr (kF32) {
                __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out) + (int64_t)row * ldo + col;
#pragma unroll
                for (int pl = 0; pl < 3; ++pl) {
                  store16<__nv_bfloat16>(out + pl * p.stride, v);
#pragma unroll
                  for (int j = 0; j < 16; ++j)
                    v[j] = __fsub_rn(v[j], __bfloat162float(__float2bfloat16_rn(v[j])));
                }
              } else {
                store16<T>(static_cast<T *>(p.out) + (int64_t)row * ldo + col, v);
              }
            }
          }
        }
      };
      // kStore, rows that begin anywhere: a chunk through shared memory, so that a store writes 32 neighbouring columns of a row.
      auto flush = [&](int ci) {
        if constexpr (kOut == Out::kStore) {
          if (vec && !staged)
            return;
          if (staged) { // eight lanes a row: 128 bytes of four rows a store
            __syncwarp();
            const int c = n0 + 32 * part + 32 * kParts * ci + 4 * (lane & 7);
            float *out = static_cast<float *>(p.out) + out0 + (int64_t)(row_base + (lane >> 3)) * ldo + c;
            float4 f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = 4 * i + (lane >> 3);
              f[i] = *reinterpret_cast<const float4 *>(stg + r * 32 + ((4 * (lane & 7)) ^ (r & 7) * 4));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i, out += 4 * ldo)
              if (row_base + 4 * i + (lane >> 3) < M) {
                if (c + 4 <= N)
                  *reinterpret_cast<float4 *>(out) = f[i];
                else
                  for (int j = 0; c + j < N; ++j)
                    out[j] = j == 0 ? f[i].x : j == 1 ? f[i].y : f[i].z;
              }
            return;
          }
          const int col0 = n0 + 32 * part + 32 * kParts * ci;
          __syncwarp();
          const int rows_here = M - row_base < 32 ? M - row_base : 32;
          const int64_t off = out0 + (int64_t)row_base * ldo + col0 + lane;
          if (col0 + lane >= N)
            return;
          auto write = [&](auto *out) {
            using O = std::remove_pointer_t<decltype(out)>;
            auto at = [&](int i) { return stg[i * S::kPitch + (kF32 ? lane : lane ^ i)]; };
            if (!kLong && !accum && rows_here == 32) { // (eight reads, then eight stores: in turn each store would wait for its read)
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                float f[8];
#pragma unroll
                for (int u = 0; u < 8; ++u)
                  f[u] = at(i + u);
#pragma unroll
                for (int u = 0; u < 8; ++u)
                  out[(i + u) * ldo] = from_f32<O>(f[u]);
              }
            } else if (accum) {
#pragma unroll 8
              for (int i = 0; i < rows_here; ++i, out += ldo)
                *out = from_f32<O>(to_f32(*out) + at(i));
            } else {
#pragma unroll 8
              for (int i = 0; i < rows_here; ++i, out += ldo)
                *out = from_f32<O>(at(i));
            }
          };
          if (out_f32)
            write(static_cast<float *>(p.out) + off);
          else
            write(static_cast<T *>(p.out) + off);
        }
      };
      auto wait_for = [&](int buf) {
        const bool got = ptx::mbar_wait(tmem_full + buf, (uint32_t)(local >> 1) & 1u, abort_flag);
        if (!__all_sync(0xffffffffu, got)) {
          if (lane == 0)
            gave_up(kStatusEpilogueTimeout);
          ok = false;
        }
        ptx::tc_fence_after_sync();
      };
      auto release = [&](int buf) {
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (kPair)
            ptx::mbar_arrive_cluster(ptx::map_to_cta(ptx::smem_u32(tmem_empty + buf), 0));
          else
            ptx::mbar_arrive(tmem_empty + buf);
        }
      };
      if constexpr (kLong) {
        // every chunk of K to registers, the last one too: tensor memory is free again while the sums are worked on
        for (int kc = 0; kc < chunks; ++kc, ++local) {
          const int buf = local & 1;
          wait_for(buf);
          if (!ok)
            break;
#pragma unroll
          for (int i = 0; i < 2 * kMyChunks; ++i) {
            const int c = 32 * part + 32 * kParts * (i / 2) + 16 * (i & 1);
            if (n0 + c >= N)
              break;
            uint32_t r[16];
            ptx::tmem_ld_32x16(lanes + (uint32_t)(buf * BN + c), r);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j)
              acc[i][j] = kc == 0 ? __uint_as_float(r[j]) : __fadd_rn(acc[i][j], __uint_as_float(r[j]));
          }
          release(buf);
        }
        if (ok && row_base < M) {
#pragma unroll
          for (int ci = 0; ci < kMyChunks; ++ci) {
            if (n0 + 32 * part + 32 * kParts * ci >= N)
              break;
            __syncwarp(); // (the staged chunk before has been read)
            finish(ci, 0, acc[2 * ci]);
            finish(ci, 1, acc[2 * ci + 1]);
            flush(ci);
          }
        }
      } else {
        const int buf = local & 1;
        wait_for(buf);
        if (!ok)
          break;
#pragma unroll
        for (int ci = 0; ci < kMyChunks; ++ci) {
          const int c = 32 * part + 32 * kParts * ci;
          if (n0 + c >= N || row_base >= M)
            break;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            __syncwarp(); // (the staged chunk before has been read, and the load is the whole warp's)
            uint32_t r[16];
            ptx::tmem_ld_32x16(lanes + (uint32_t)(buf * BN + c + 16 * h), r);
            ptx::tmem_ld_wait();
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j)
              v[j] = __uint_as_float(r[j]);
            finish(ci, h, v);
          }
          flush(ci);
        }
        release(buf);
        ++local;
      }
      if constexpr (kOut == Out::kSums)
        if (ok && row_ok)
          rows.partial[(int64_t)row * rows.tiles + n0 / BN * kParts + part] = make_float2(t.m, t.s);
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
  if (kPair)
    ptx::cluster_sync(); // neither CTA leaves while its peer may still signal its barriers
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    if (kPair)
      ptx::tmem_dealloc_pair(tmem_base, kTmemCols);
    else
      ptx::tmem_dealloc(tmem_base, kTmemCols);
  }
}

// An operand in memory: `planes` matrices [rows][pitch] of 16-bit values, plane_rows rows apart; 16-byte aligned, pitch a
// multiple of 8.
struct Operand {
  const void *p;
  int64_t rows, cols, pitch;
  int planes;
  int64_t plane_rows;
};
// Boxes of 64 values by box_rows rows of memory. The copy engine takes 4 to 6 cycles a row of a box, rows outside the matrix
// included, so boxes are as high as the matrix where that is low: of 8 rows of x a box of 128 took most of a tile's time
// ([8, 1792] . [1792, 109056] bf16 184 us). What the MMAs read beyond a box is of rows that no one stores.
inline int loss_operand_map(CUtensorMap *map, const Operand &o, int box_rows) {
  const uint64_t dims[3] = {(uint64_t)o.cols, (uint64_t)o.rows, (uint64_t)o.planes};
  const uint64_t strides[2] = {(uint64_t)o.pitch * 2, (uint64_t)(o.pitch * o.plane_rows) * 2};
  const uint32_t box[3] = {64, (uint32_t)box_rows, 1};
  return encode_tiled(map, 0, 3, o.p, dims, strides, box, nullptr, 128);
}

// 16 bits: 96 steps (an error of 1.4e-6 of the result's RMS, and three times that after a thousand); fp32: a K block, whose
// last four steps are the only ones on a large accumulator
template <typename T> constexpr int loss_chunk() { return std::is_same<T, float>::value ? 1 : 24; }
// Whether a product's K goes through tensor memory in more than one chunk. Of dx and dW in fp32 two K blocks are one, without the
// sums in registers (dW of 65 to 128 rows, which its stores bound).
template <typename T, Out kOut = Out::kStore> bool loss_is_long(int64_t kblocks) {
  return kblocks > (std::is_same<T, float>::value && kOut == Out::kStore ? 2 : loss_chunk<T>());
}
// The maxima and sums that kSums leaves of a row.
template <typename T> int loss_sum_tiles(int64_t classes, int64_t kblocks, bool pair) {
  return (int)(pair ? (classes + 255) / 256 * (loss_is_long<T>(kblocks) || std::is_same<T, float>::value ? 2 : 4)
                    : (classes + 63) / 64 * 2);
}

template <typename T, bool kPair, bool kLong, Out kOut, bool kSplit = false>
inline int launch_loss_gemm(Products prob, const Operand *a, const Operand *b, cudaStream_t st) {
  constexpr int PL = std::is_same<T, float>::value ? 3 : 1;
  using S = LossShape<PL, kPair, kLong, kSplit>;
  auto kernel = loss_gemm_kernel<T, kPair, kLong, kOut, kSplit>;
  static std::atomic<bool> configured[64]{};
  int dev = 0;
  NB_CUDA(cudaGetDevice(&dev));
  if (!configured[dev & 63]) {
    NB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
    configured[dev & 63] = true;
  }
  Operand oa[kMaxProducts], ob[kMaxProducts];
  for (int i = 0; i < prob.count; ++i) {
    oa[i] = a[i], ob[i] = kSplit ? a[i] : b[i];
    if (prob.p[i].splits <= 1)
      prob.p[i].splits = 1, prob.p[i].split_blocks = prob.p[i].kblocks;
  }
  if (prob.count == 2 && prob.p[0].split_blocks < prob.p[1].split_blocks) { // the product with the longer tiles first
    std::swap(prob.p[0], prob.p[1]);
    std::swap(oa[0], oa[1]);
    std::swap(ob[0], ob[1]);
  }
  CUtensorMap ma[2], mb[2];
  int64_t tiles[2] = {0, 0}, cost[2] = {1, 1};
  for (int i = 0; i < prob.count; ++i) {
    Product &p = prob.p[i];
    p.m_tiles = (p.M + S::kTileRows - 1) / S::kTileRows;
    p.n_tiles = (p.N + S::kTileCols - 1) / S::kTileCols;
    tiles[i] = (int64_t)p.m_tiles * p.n_tiles * p.splits;
    cost[i] = loss_tile_cycles(p.split_blocks, kPair);
    p.steps = p.kblocks == 1 ? (p.K + 15) / 16 : 4;
    const int a_rows = p.a_mn ? 16 * p.steps : p.M < kTileM ? (p.M + 7) / 8 * 8 : kTileM;
    const int b_rows = p.b_mn ? 16 * p.steps : S::kCtaCols;
    p.tx_bytes = PL * kRowBytes * ((p.a_mn ? kTileM / 64 : 1) * a_rows + (kSplit ? 0 : p.b_mn ? S::kCtaCols / 64 : 1) * b_rows);
    NB_TRY(loss_operand_map(&ma[i], oa[i], a_rows));
    if (kSplit)
      mb[i] = ma[i];
    else
      NB_TRY(loss_operand_map(&mb[i], ob[i], b_rows));
  }
  NB_CHECK(tiles[0] + tiles[1] < (1ll << 31), NB200_EVALUE, "too many rows and classes");
  if (prob.count == 1)
    ma[1] = ma[0], mb[1] = mb[0];
  constexpr int kCtas = kPair ? 2 : 1;
  const int64_t units = std::min<int64_t>(sm_count() / kCtas, tiles[0] + tiles[1]);
  prob.extra_tiles = (int)extra_tiles(tiles[0], tiles[1], cost[0], cost[1], units);
  prob.chunk = kLong ? loss_chunk<T>() : 1 << 20;
  int *status = nullptr;
  NB_TRY(device_status_word(&status));
  NB_CUDA(launch_clusters(kernel, (unsigned)(kCtas * units), kCtas, S::kThreads, S::kSmem, st, ma[0], mb[0], ma[1], mb[1], prob,
                          status));
  return NB200_OK;
}
template <typename T, Out kOut>
int run_loss_gemm(bool pair, const Products &prob, const Operand *a, const Operand *b, cudaStream_t st) {
  bool is_long = false;
  for (int i = 0; i < prob.count; ++i)
    is_long = is_long || loss_is_long<T, kOut>(prob.p[i].splits > 1 ? prob.p[i].split_blocks : prob.p[i].kblocks);
  if (!is_long)
    return (pair ? launch_loss_gemm<T, true, false, kOut> : launch_loss_gemm<T, false, false, kOut>)(prob, a, b, st);
  return (pair ? launch_loss_gemm<T, true, true, kOut> : launch_loss_gemm<T, false, true, kOut>)(prob, a, b, st);
}

// The same in fp32 with B as it lies: [rows, cols] of a matrix whose rows are ld values apart.
template <Out kOut>
int run_split_gemm(Products prob, const Operand &a, const float *b, int64_t rows, int64_t cols, int64_t ld, cudaStream_t st) {
  Product &p = prob.p[0];
  p.b = b, p.b_rows = rows, p.b_cols = cols, p.b_ld = ld;
  p.b_pairs = ld % 2 == 0 && (reinterpret_cast<uintptr_t>(b) & 7) == 0;
  return launch_loss_gemm<float, false, true, kOut, true>(prob, &a, nullptr, st);
}

} // namespace nb200
