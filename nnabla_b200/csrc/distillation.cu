// Distillation from a teacher of which each row's K best classes and their logits are known.
//
//   p = softmax(teacher / tau) over the row's entries (class >= 0), q = softmax(x / tau) over all classes
//   loss = tau^2 sum_k p_k (log p_k - log q_k)
//   dx_v = tau (q_v [the row has an entry] - sum of p_k over the entries k of class v) dloss
//
// HBM bound: the forward pass reads x once, with the running maximum and sum of the softmax; with those two kept, the
// gradient is one pass that reads x and writes dx, and then corrects the few classes that the teacher names. Differences to
// the maximum are taken before anything is scaled: a row masked with the type's lowest value overflows nowhere.
#include <algorithm>

#include "pdl.cuh"
#include "softmax_sums.cuh"

namespace nb200 {
namespace {

constexpr int kMaxEntries = 1024;

// The row's teacher, by one warp: each lane's entries are k = lane, lane + 32, ... The first kHeld of them stay in registers, on
// their way while the row of x is read. An entry is one with a class that is not negative.
constexpr int kHeld = 4;
template <typename T, typename I> struct Entries {
  const I *index;
  const T *teacher;
  int best, lane;
  I c[kHeld];
  T t[kHeld];
  __device__ __forceinline__ Entries(const I *index_, const T *teacher_, int best_, int lane_)
      : index(index_), teacher(teacher_), best(best_), lane(lane_) {
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      c[u] = -1;
      if (lane + 32 * u < best) {
        c[u] = index[lane + 32 * u];
        t[u] = teacher[lane + 32 * u];
      }
    }
  }
  // f(class, logit, u) for this lane's entries; u: the held one's number, kHeld for the others
  template <typename F> __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int u = 0; u < kHeld; ++u)
      if (c[u] >= 0)
        f((int64_t)c[u], to_f32(t[u]), u);
    for (int k = lane + 32 * kHeld; k < best; k += 32)
      if (index[k] >= 0)
        f((int64_t)index[k], to_f32(teacher[k]), kHeld);
  }
  __device__ __forceinline__ MaxSum sums(float scale) const {
    MaxSum s{-INFINITY, 0.0f};
    float top = -INFINITY;
    bool nan = false;
    each([&](int64_t, float v, int) {
      top = fmaxf(top, v);
      nan |= v != v;
    });
    top = __any_sync(0xffffffffu, nan) ? NAN : warp_max(top);
    s.m = top;
    const float base = top == -INFINITY ? 0.0f : top;
    each([&](int64_t, float v, int) { s.s += ex2((v - base) * scale); });
    s.s = warp_sum(s.s);
    return s;
  }
};

// [start, start + n) of x cut into values before the first 16-byte boundary, whole 16-byte packs, and the rest.
template <typename T> struct Run {
  const T *head, *body, *tail;
  int heads, tails;
  int64_t packs;
  __device__ __forceinline__ Run(const T *start, int64_t n) {
    constexpr int V = kPackOf<T>;
    int h = (int)((16 - (reinterpret_cast<uintptr_t>(start) & 15)) & 15) / (int)sizeof(T);
    heads = h < n ? h : (int)n;
    head = start;
    body = start + heads;
    packs = (n - heads) / V;
    tail = body + packs * V;
    tails = (int)(n - heads - packs * V);
  }
};

// Measured at [4096, 128000] bf16, 64 entries a row: forward 186 us (5.7 TB/s), gradient 354 us (5.9 TB/s; 624 with a block a piece
// of 8192 classes, each of which waited for the teacher's sums).
constexpr int kSumThreads = 256;

// One row a cluster of blocks (one block where the rows are many). stat: the row's maximum, and log sum exp((x - maximum) / tau).
template <typename T, typename I>
__global__ void __launch_bounds__(kSumThreads, 4) distill_forward_kernel(const T *__restrict__ x, const I *__restrict__ index,
                                                              const T *__restrict__ teacher, float *__restrict__ loss,
                                                              float2 *__restrict__ stat, int64_t classes, int best,
                                                              float tau, int parts) {
  constexpr int V = kPackOf<T>;
  __shared__ float shared_m[16], shared_s[16];
  __shared__ float whole[2];
  pdl_wait();
  pdl_trigger();
  const int64_t row = blockIdx.x / parts;
  const int part = blockIdx.x - (int)row * parts;
  const int64_t each = ((classes + parts - 1) / parts + V - 1) / V * V;
  const int64_t c0 = part * each < classes ? part * each : classes, c1 = c0 + each < classes ? c0 + each : classes;
  const T *xr = x + row * classes;
  const float scale = kLog2e / tau;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const Run<T> run(xr + c0, c1 - c0);
  // the teacher's entries, and x there, for the first block's first warp (none for the others)
  const Entries<T, I> entries(index + row * best, teacher + row * best, part == 0 && warp == 0 ? best : 0, lane);
  T named[kHeld];
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    if (entries.c[u] >= 0 && (int64_t)entries.c[u] < classes)
      named[u] = xr[entries.c[u]];
  float m = -INFINITY, s = 0.0f;
  auto add = [&](auto &v, int n) {
    float top = m;
#pragma unroll
    for (int j = 0; j < n; ++j)
      top = fmaxf(top, v[j]);
    const float base = top == -INFINITY ? 0.0f : top;
    s *= ex2((m - base) * scale);
#pragma unroll
    for (int j = 0; j < n; ++j)
      s += ex2((v[j] - base) * scale);
    m = top;
  };
  const int64_t step = blockDim.x;
  int64_t i = threadIdx.x;
  for (; i + 3 * step < run.packs; i += 4 * step) {
    Pack<T, V> p[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      p[u] = load_pack_stream<T, V>(run.body + (i + u * step) * V);
    float v[4 * V];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j)
        v[u * V + j] = p[u].f(j);
    add(v, 4 * V);
  }
  for (; i < run.packs; i += step) {
    const Pack<T, V> p = load_pack_stream<T, V>(run.body + i * V);
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j)
      v[j] = p.f(j);
    add(v, V);
  }
  if ((int)threadIdx.x < run.heads + run.tails) {
    float v[1] = {to_f32((int)threadIdx.x < run.heads ? run.head[threadIdx.x] : run.tail[threadIdx.x - run.heads])};
    add(v, 1);
  }
  MaxSum t = warp_join({m, s}, scale);
  if (lane == 0)
    shared_m[warp] = t.m, shared_s[warp] = t.s;
  __syncthreads();
  if (warp == 0) {
    t = warp_join(lane < warps ? MaxSum{shared_m[lane], shared_s[lane]} : MaxSum{-INFINITY, 0.0f}, scale);
    if (lane == 0)
      whole[0] = t.m, whole[1] = t.s;
  }
  if (parts > 1) {
    cluster_barrier();
    if (part == 0 && warp == 0) {
      MaxSum o{-INFINITY, 0.0f};
      if (lane < parts) {
        uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(whole)), theirs;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(theirs) : "r"(mine), "r"(lane));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.m) : "r"(theirs) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.s) : "r"(theirs + 4u) : "memory");
      }
      t = warp_join(o, scale);
    }
  }
  if (part == 0 && warp == 0) {
    const float log_sum = log2f(t.s) * kLn2;
    const MaxSum p = entries.sums(scale);
    // In 64 bits, and divided by the shares' own sum: a class that the student masks with the type's lowest value and the
    // teacher names gives a loss next to the largest float.
    double sum = 0.0, mass = 0.0;
    const double per = 1.0 / (double)tau;
    if (p.m != -INFINITY) {
      const double log_mass = log2f(p.s) * kLn2;
      entries.each([&](int64_t c, float v, int u) {
        const float d = v - p.m, share = ex2(d * scale);
        mass += share;
        if (c >= classes) {
          sum = NAN;
        } else if (!(share == 0.0f)) {
          float at = 0.0f;
#pragma unroll
          for (int i = 0; i < kHeld; ++i)
            at = u == i ? to_f32(named[i]) : at;
          if (u == kHeld)
            at = to_f32(xr[c]);
          sum += share * ((d * per - log_mass) - (((double)at - t.m) * per - log_sum));
        }
      });
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      mass += __shfl_xor_sync(0xffffffffu, mass, o);
    }
    if (p.m != -INFINITY)
      sum /= mass;
    if (lane == 0) {
      loss[row] = (float)(sum * tau * tau);
      stat[row] = make_float2(t.m, log_sum);
    }
  }
  if (parts > 1) // no block leaves while another may still read its sums
    cluster_barrier();
}

constexpr int kGradThreads = 256, kGradPacks = 4;

// dx (+)= gradient, a part of a row a block. Warp 0 takes the teacher's sums and lists the entries whose class lies in the
// part; those classes' gradients are made first, from x as it is before anything is written (dx may be x), and stored last, by
// the first of the entries that name them. The rest is one stream.
template <typename T, typename I>
__global__ void __launch_bounds__(kGradThreads, 4) distill_backward_kernel(
    const T *x, const I *__restrict__ index, const T *__restrict__ teacher, const float2 *__restrict__ stat,
    const float *__restrict__ dloss, T *dx, int64_t classes, int best, float tau, int parts, bool accum, bool keep) {
  constexpr int V = kPackOf<T>;
  __shared__ int at[kMaxEntries];
  __shared__ float share[kMaxEntries];
  __shared__ int entries;
  __shared__ float weight; // 1 where the row has an entry, 0 where it has none, NaN where an entry's class does not exist
  pdl_wait();
  pdl_trigger();
  const int64_t row = blockIdx.x / parts;
  const int part = blockIdx.x - (int)row * parts;
  const T *xr = x + row * classes;
  T *out = dx + row * classes;
  // parts begin at 16-byte boundaries of x but for the row's first
  const int64_t lead = (int64_t)(((16 - (reinterpret_cast<uintptr_t>(xr) & 15)) & 15) / sizeof(T));
  const int64_t each = ((classes + parts - 1) / parts + V - 1) / V * V;
  int64_t c0 = part == 0 ? 0 : lead + part * each, c1 = lead + (part + 1) * each;
  c1 = c1 < classes && part + 1 < parts ? c1 : classes;
  c0 = c0 < c1 ? c0 : c1;
  const Run<T> run(xr + c0, c1 - c0);
  // the first loads of the stream are on their way while the entries are looked at
  Pack<T, V> ahead[kGradPacks];
#pragma unroll
  for (int u = 0; u < kGradPacks; ++u)
    if (threadIdx.x + u * kGradThreads < run.packs)
      ahead[u] = load_pack_stream<T, V>(run.body + (threadIdx.x + u * kGradThreads) * V);
  const float scale = kLog2e / tau, d = dloss[row] * tau, top = stat[row].x, log2_sum = stat[row].y * kLog2e;
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    const Entries<T, I> all(index + row * best, teacher + row * best, best, lane);
    const MaxSum t = all.sums(scale);
    int n = 0;
    bool bad = false;
    if (t.m != -INFINITY) {
      const float log2_p = log2f(t.s);
      for (int k0 = 0; k0 < best; k0 += 32) {
        const int k = k0 + lane;
        int64_t c = -1;
        float v = 0.0f;
        if (k0 < 32 * kHeld) {
#pragma unroll
          for (int u = 0; u < kHeld; ++u)
            if (k0 == 32 * u && all.c[u] >= 0)
              c = all.c[u], v = to_f32(all.t[u]);
        } else if (k < best) {
          c = (int64_t)all.index[k], v = to_f32(all.teacher[k]);
        }
        bad |= c >= classes;
        const bool here = c >= c0 && c < c1;
        const unsigned found = __ballot_sync(0xffffffffu, here);
        if (here) {
          const int to = n + __popc(found & ((1u << lane) - 1u));
          at[to] = (int)(c - c0);
          share[to] = ex2(fmaf(v - t.m, scale, -log2_p));
        }
        n += __popc(found);
      }
    }
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) {
      entries = n;
      weight = bad ? NAN : (t.m == -INFINITY ? 0.0f : 1.0f);
    }
  }
  __syncthreads();
  const int n = entries;
  const float factor = d * weight;
  const bool dead = weight == 0.0f;
  auto q = [&](float v) { return ex2(fmaf(v - top, scale, -log2_sum)); };
  auto value = [&](float v) { return dead ? 0.0f : q(v) * factor; };
  float fixed[kMaxEntries / kGradThreads];
  unsigned first = 0; // bit u: entry threadIdx.x + u * kGradThreads is the first that names its class
#pragma unroll
  for (int u = 0; u < kMaxEntries / kGradThreads; ++u) {
    const int i = threadIdx.x + u * kGradThreads;
    if (i >= n)
      continue;
    float sum = 0.0f;
    bool only = true;
#pragma unroll 8
    for (int j = 0; j < n; ++j) {
      const bool same = at[j] == at[i];
      only &= !same || j >= i;
      sum += same ? share[j] : 0.0f;
    }
    if (only) {
      first |= 1u << u;
      fixed[u] = (q(to_f32(xr[c0 + at[i]])) - sum) * factor;
      if (accum)
        fixed[u] += to_f32(out[c0 + at[i]]);
    }
  }
  if (n > 0)
    __syncthreads();
  auto store = [&](T *to, const Pack<T, V> &p) {
    float o[V];
#pragma unroll
    for (int j = 0; j < V; ++j)
      o[j] = value(p.f(j));
    if ((reinterpret_cast<uintptr_t>(to) & 15) == 0) {
      if (accum) {
        const Pack<T, V> old = load_pack<T, V>(to);
#pragma unroll
        for (int j = 0; j < V; ++j)
          o[j] += old.f(j);
      }
      store_pack<T, V>(to, o, keep);
    } else { // (dx lies differently from x)
#pragma unroll
      for (int j = 0; j < V; ++j)
        to[j] = from_f32<T>(accum ? o[j] + to_f32(to[j]) : o[j]);
    }
  };
  T *body = out + (run.body - xr);
#pragma unroll
  for (int u = 0; u < kGradPacks; ++u)
    if (threadIdx.x + u * kGradThreads < run.packs)
      store(body + (threadIdx.x + u * kGradThreads) * V, ahead[u]);
  int64_t i = threadIdx.x + kGradPacks * kGradThreads;
  for (; i + (kGradPacks - 1) * kGradThreads < run.packs; i += kGradPacks * kGradThreads) {
    Pack<T, V> p[kGradPacks];
#pragma unroll
    for (int u = 0; u < kGradPacks; ++u)
      p[u] = load_pack_stream<T, V>(run.body + (i + u * kGradThreads) * V);
#pragma unroll
    for (int u = 0; u < kGradPacks; ++u)
      store(body + (i + u * kGradThreads) * V, p[u]);
  }
  for (; i < run.packs; i += kGradThreads)
    store(body + i * V, load_pack_stream<T, V>(run.body + i * V));
  if ((int)threadIdx.x < run.heads + run.tails) {
    const T *from = (int)threadIdx.x < run.heads ? run.head + threadIdx.x : run.tail + (threadIdx.x - run.heads);
    T *to = out + (from - xr);
    const float o = value(to_f32(*from));
    *to = from_f32<T>(accum ? o + to_f32(*to) : o);
  }
  if (n == 0)
    return;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kMaxEntries / kGradThreads; ++u)
    if (first >> u & 1)
      out[c0 + at[threadIdx.x + u * kGradThreads]] = from_f32<T>(fixed[u]);
}

int check(int64_t rows, int64_t classes, int best, float temperature, int index_bytes) {
  NB_CHECK(rows >= 0 && rows < (1ll << 24), NB200_EVALUE, "%lld rows", (long long)rows);
  NB_CHECK(classes > 0 && classes < (1ll << 24), NB200_EVALUE, "%lld classes outside [1, 2^24)", (long long)classes);
  NB_CHECK(best >= 1 && best <= kMaxEntries, NB200_EVALUE, "%d entries a row outside [1, %d]", best, kMaxEntries);
  // (the inverse of a smaller one is infinite)
  NB_CHECK(temperature >= 1.17549435e-38f && temperature < INFINITY, NB200_EVALUE, "temperature = %g outside [2^-126, infinity)",
           temperature);
  NB_CHECK(index_bytes == 4 || index_bytes == 8, NB200_EVALUE, "the classes are 4 or 8 byte integers, not %d", index_bytes);
  return NB200_OK;
}

template <typename T, typename I>
int forward(const T *x, const I *index, const T *teacher, float *loss, float *stat, int64_t rows, int64_t classes,
            int best, float tau, cudaStream_t st) {
  // few long rows go to clusters
  const int64_t packs = (classes + kPackOf<T> - 1) / kPackOf<T>;
  int parts = 1;
  while (parts < 8 && rows * parts < 2 * sm_count() && packs >= 512 * parts)
    parts *= 2;
  const int threads = packs <= 256 ? 128 : kSumThreads;
  NB_CUDA(launch_clusters(distill_forward_kernel<T, I>, (unsigned)(rows * parts), parts, threads, 0, st, x, index, teacher, loss,
                          reinterpret_cast<float2 *>(stat), classes, best, tau, parts));
  return NB200_OK;
}

template <typename T, typename I>
int backward(const T *x, const I *index, const T *teacher, const float *stat, const float *dloss, T *dx, int64_t rows,
             int64_t classes, int best, float tau, bool accum, cudaStream_t st) {
  // a row a block, or in parts, of one round of its loads at least, until the blocks fill the SMs
  const int64_t packs = (classes + kPackOf<T> - 1) / kPackOf<T>, most = (packs + kGradThreads * kGradPacks - 1) / (kGradThreads * kGradPacks);
  const int64_t parts = std::min<int64_t>(most, (8 * sm_count() + rows - 1) / rows);
  const bool keep = (size_t)rows * classes * sizeof(T) <= kKeepBytes;
  NB_CUDA(launch_dependent(distill_backward_kernel<T, I>, dim3((unsigned)(rows * parts)), dim3(kGradThreads), 0, st, x,
                           index, teacher, reinterpret_cast<const float2 *>(stat), dloss, dx, classes, best, tau, (int)parts,
                           accum, keep));
  return NB200_OK;
}

} // namespace
} // namespace nb200

using namespace nb200;

extern "C" int nb200_top_k_distillation(const void *x, const void *index, const void *teacher, float *loss, float *stat,
                                        int64_t rows, int64_t classes, int best, float temperature, int type,
                                        int index_bytes, void *stream) {
  NB_TRY(check(rows, classes, best, temperature, index_bytes));
  if (rows == 0)
    return NB200_OK;
  NB_CHECK(x && index && teacher && loss && stat, NB200_EVALUE, "null data pointer");
  NB_CHECK((reinterpret_cast<uintptr_t>(stat) & 7) == 0, NB200_EVALUE, "stat holds pairs: 8-byte aligned");
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    auto run = [&](auto i) {
      using I = decltype(i);
      return forward<T, I>(static_cast<const T *>(x), static_cast<const I *>(index), static_cast<const T *>(teacher), loss,
                           stat, rows, classes, best, temperature, as_stream(stream));
    };
    return index_bytes == 8 ? run(int64_t{}) : run(int32_t{});
  });
}

extern "C" int nb200_top_k_distillation_backward(const void *x, const void *index, const void *teacher,
                                                 const float *stat, const float *dloss, void *dx, int64_t rows,
                                                 int64_t classes, int best, float temperature, int type, int index_bytes,
                                                 int accum, void *stream) {
  NB_TRY(check(rows, classes, best, temperature, index_bytes));
  if (rows == 0)
    return NB200_OK;
  NB_CHECK(x && index && teacher && stat && dloss && dx, NB200_EVALUE, "null data pointer");
  NB_CHECK((reinterpret_cast<uintptr_t>(stat) & 7) == 0, NB200_EVALUE, "stat holds pairs: 8-byte aligned");
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    auto run = [&](auto i) {
      using I = decltype(i);
      return backward<T, I>(static_cast<const T *>(x), static_cast<const I *>(index), static_cast<const T *>(teacher),
                            stat, dloss, static_cast<T *>(dx), rows, classes, best, temperature, accum != 0,
                            as_stream(stream));
    };
    return index_bytes == 8 ? run(int64_t{}) : run(int32_t{});
  });
}
