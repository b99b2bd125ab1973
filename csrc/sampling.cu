// One token a row from its logits: temperature, top-k, top-p, min-p, and the draw from a given uniform number.
//
//   w_i = 2^((l_i - max l) log2(e) / T);  order by (logit descending, index ascending);  the first k stay;  of these those with (weight before them) < p Z, Z the sum
//   of the first k;  of these those with w >= min_p;  the token is the first index, in vocabulary order, whose cumulative weight exceeds u times the sum of what stays.
//
// A token is a whole number: what decides it is computed in 64 bits (a relative error of 1e-7 in the sums would move one draw in some thousand over a flat
// vocabulary).  2^t is the table method of P. T. P. Tang (1989): 2^(k/32) from a table that lies across a warp's lanes, times a polynomial of degree 5 in the rest.
//
// A cluster of CTAs holds a row in shared memory: it is read once (with many long rows fewer CTAs read it again, from L2, four logits a lane: one a lane took 363 us for 280).  Every cut is a place in the one order (key, index), found by counts over 2048 bins and, where weights
// decide, by exact sums above, in and below the bin that the counts suggest.  What is left of a bin goes into a list that one CTA sorts; equal logits beyond the list
// are cut by their indices alone.  What top-k leaves of up to 1024 is listed whole, and one CTA cuts and draws among it, by bins of whole-number weights; for small k
// the k-th largest of the threads' maxima, which bounds the k-th logit from below, saves the counts over all.  Compiled without fast math.
//
// Bound: no pipe, but latencies in the chain of some ten steps in which a row's CTAs wait for one another, the longest by mass the counts (atomics in shared memory, 5 us for
// 16384 logits) and the weights (8 to 11 us).  128 rows of 262144 by mass: 272 us, issue slots 56 % used, the pipe for 64 bits 13 %, memory 18 %; warps wait for fixed
// latencies, loads from L2 and barriers.  256 of 50304 in fp32, no filter: 39 us, 52, 28 and 14 %.  33 rows of 248320 in bf16, settings of all kinds: 58; 1 row of 151936,
// top-k 50 and top-p: 12, 9 of them the host's.
#include <cooperative_groups.h>

#include <type_traits>

#include "common.cuh"
#include "per_device.h"

namespace tyr {
namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 2048, kSampleList = 1024, kSampleCluster = 16;
constexpr int kSampleMost = 2048;                                          // of a list that holds all that top-k leaves
constexpr int kSampleScratch = 3 * kSampleMost * 8;                        // bytes that CTA 0 needs beside it, where its logits were
constexpr int kSampleSlice = 16384, kSampleLargest = 40960;                // logits that a CTA holds: with two of them on an SM, and at most
constexpr int kSampleRead = 65536;                                         // logits of a CTA that reads them anew for every pass

struct SampleArgs {
  const void* logits;                    // [rows, V], row stride below
  const void* draws;                     // [rows] fp32 or fp64
  const float *temperature, *top_p, *min_p;      // [rows] (null: the numbers below)
  const int* top_k;
  long long* token;
  long long row;
  double t, p, m;
  int rows, V, slice, draws64, k, pad;
};
static_assert(sizeof(SampleArgs) == 112, "as ops/sampling.py packs it");

struct Place { uint32_t key, index; };                                     // what comes no later in the order stays

__device__ __forceinline__ uint32_t key_of(float x) {                      // 0: never chosen (-inf, NaN, behind the row)
  const uint32_t b = __float_as_uint(x);
  if (!(x > -INFINITY)) return 0u;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ bool stays(uint32_t key, uint32_t index, Place c) { return key > c.key || (key == c.key && index <= c.index); }

__device__ __forceinline__ float load_logit(const float* p) { return __ldg(p); }
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(__ldg(p)); }
__device__ __forceinline__ float load_logit(const __half* p) { return __half2float(__ldg(p)); }
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_scan_d(double v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

struct Weights {                         // 2^((x - top) c), all lanes of a warp together; 2^-900, next to nothing, where it would be less and for -inf
  double table, top, c;
  __device__ __forceinline__ double operator()(float x) const {
    const double far = (static_cast<double>(x) - top) * c;                  // never positive: as unsigned numbers, the larger the further
    const double t = __hiloint2double(static_cast<int>(min(static_cast<uint32_t>(__double2hiint(far)), 0xC08C2000u)), __double2loint(far));
    constexpr double kMagic = 211106232532992.0;                           // 1.5 * 2^47: its last place is 2^-5
    const double r = t + kMagic, f = t - (r - kMagic);
    const int k = __double2loint(r);
    // ln2^i / i!
    const double e = fma(f, fma(f, fma(f, fma(f, fma(f, 1.3333558146428443e-3, 9.618129107628477e-3), 5.550410866482158e-2), 2.402265069591007e-1), 6.931471805599453e-1), 1.0);
    const double w = __shfl_sync(0xffffffffu, table, k) * e;
    return __hiloint2double(__double2hiint(w) + ((k >> 5) << 20), __double2loint(w));
  }
};

struct Partial { double above, in, all; uint32_t count, low, high, pad; };

struct SampleShared {
  union {
    struct { uint32_t bins[kSampleBins], total[kSampleBins]; };
    unsigned long long mass[kSampleBins];
  };
  unsigned long long list[kSampleList], fixed[kSampleList];                // items and their weights
  double warp_sums[kSampleWarps], cta_sums[kSampleCluster], run_sums[kSampleRead / kSampleThreads];
  Partial part[2][kSampleCluster], warp_part[kSampleWarps];
  double warp_above[kSampleWarps];                                         // of a warp's logits above the bin of the cut
  float tops[kSampleCluster], warp_top[kSampleWarps];
  unsigned long long own[kSampleList];                                     // of the bin of the cut, this CTA's
  unsigned long long best, bests[kSampleCluster];
  uint32_t scan[kSampleWarps], listed, collected, counts[kSampleCluster * kSampleWarps];
  double scan_d[kSampleWarps];
  Place cut;
  unsigned long long scan_u[kSampleWarps], base;
  int found, flag;
};

__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* s, uint32_t& total) {      // inclusive
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) s[warp] = v;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kSampleWarps; ++i) {
    if (i < warp) before += s[i];
    total += s[i];
  }
  return v + before;
}
__device__ __forceinline__ double block_scan_d(double v, double* s, double& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_scan_d(v, lane);
  __syncthreads();
  if (lane == 31) s[warp] = v;
  __syncthreads();
  double before = 0.0;
  total = 0.0;
#pragma unroll
  for (int i = 0; i < kSampleWarps; ++i) {
    if (i < warp) before += s[i];
    total += s[i];
  }
  return v + before;
}
__device__ __forceinline__ unsigned long long block_scan_u(unsigned long long v, unsigned long long* s, unsigned long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) s[warp] = v;
  __syncthreads();
  unsigned long long before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kSampleWarps; ++i) {
    if (i < warp) before += s[i];
    total += s[i];
  }
  return v + before;
}
// n different items, largest first: as many threads as there are to an item count those before it.
__device__ __forceinline__ void block_rank(unsigned long long* v, unsigned long long* to, int n) {
  const int each = n > 128 ? 2 : n > 64 ? 4 : n > 32 ? 8 : n > 16 ? 16 : 32, i = threadIdx.x / each;
  __syncthreads();
  const unsigned long long x = i < n ? v[i] : ~0ull;
  int before = 0;
  for (int j = threadIdx.x % each; j < n; j += each) before += v[j] > x;
  for (int o = 1; o < each; o <<= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if (i < n && threadIdx.x % each == 0) to[before] = x;
  __syncthreads();
  if (threadIdx.x < n) v[threadIdx.x] = to[threadIdx.x];
  __syncthreads();
}
// n items (a power of two, 64 at least), largest first: a bitonic network over two neighbouring items a thread.  Exchanges within a warp's 64 items take no shared
// memory and no barrier, which leaves one exchange in ten for 64 items more, two for 128 and so on.
__device__ __forceinline__ void block_sort(unsigned long long* v, int n) {
  __syncthreads();
  const int at = 2 * threadIdx.x;
  const bool on = at < n;                                                  // whole warps
  unsigned long long x = on ? v[at] : 0, y = on ? v[at + 1] : 0;
  for (int size = 2; size <= n; size <<= 1) {
    for (int step = size >> 1; step > 0; step >>= 1) {
      const bool down = (at & size) == 0;                                  // largest first in this run
      if (step >= 64) {
        __syncthreads();
        if (on) v[at] = x, v[at + 1] = y;
        __syncthreads();
        if (on) {
          const bool upper = (at & step) == 0;
          const unsigned long long p = v[at ^ step], q = v[(at + 1) ^ step];
          x = upper == down ? max(x, p) : min(x, p);
          y = upper == down ? max(y, q) : min(y, q);
        }
      } else if (on) {
        if (step == 1) {
          const unsigned long long p = max(x, y), q = min(x, y);
          x = down ? p : q;
          y = down ? q : p;
        } else {
          const bool upper = (at & step) == 0;
          const unsigned long long p = __shfl_xor_sync(0xffffffffu, x, step >> 1), q = __shfl_xor_sync(0xffffffffu, y, step >> 1);
          x = upper == down ? max(x, p) : min(x, p);
          y = upper == down ? max(y, q) : min(y, q);
        }
      }
    }
  }
  __syncthreads();
  if (on) v[at] = x, v[at + 1] = y;
  __syncthreads();
}

template <typename T, bool HELD>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const __grid_constant__ SampleArgs a) {
  constexpr int WARPS = kSampleWarps;
  pdl_trigger();
  cluster_arrive();                                                        // no CTA writes into another's shared memory before that one runs
  pdl_wait();
  extern __shared__ __align__(16) float s_logits[];                        // 16-byte stores and lists of 64-bit items
  __shared__ SampleShared s;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank(), row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* logits = static_cast<const T*>(a.logits) + row * a.row;
  // a CTA's slice and a warp's part of it are consecutive; a lane looks at every 32nd
  const int per_warp = a.slice / WARPS, its = per_warp / 32, base = rank * a.slice + warp * per_warp + lane;
  const auto clean = [](float v) { return v == 0.f ? 0.f : (v != v ? -INFINITY : v); };        // -0 is 0, NaN is never chosen
  float top = -INFINITY;
  {
    constexpr int VEC = 16 / sizeof(T);
    const int first = base - lane, here = max(0, min(per_warp, a.V - first));
    float* part = s_logits + warp * per_warp;
    int done = 0;
    if ((reinterpret_cast<uintptr_t>(logits + first) & 15) == 0) {
      done = here / VEC * VEC;
#pragma unroll 8
      for (int i = lane * VEC; i < done; i += 32 * VEC) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(logits + first + i));
        T v[VEC];
        *reinterpret_cast<uint4*>(v) = u;
        float f[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) top = fmaxf(top, f[e] = clean(to_float(v[e])));
#pragma unroll
        for (int e = 0; HELD && e < VEC; e += 4) *reinterpret_cast<float4*>(part + i + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
      }
    }
#pragma unroll 16
    for (int i = done + lane; i < per_warp; i += 32) {
      const float v = i < here ? clean(load_logit(logits + first + i)) : -INFINITY;
      if constexpr (HELD) part[i] = v;
      top = fmaxf(top, v);
    }
    __syncwarp();
  }
  const double T_row = a.temperature ? a.temperature[row] : a.t, p = a.top_p ? a.top_p[row] : a.p, m_row = a.min_p ? a.min_p[row] : a.m;
  const double m = m_row > 0.0 ? fmin(m_row, 1.0) : 0.0;                   // no number: no filter, as p
  const int k_row = a.top_k ? a.top_k[row] : a.k;
  float own_top = top;
  top = warp_max(top);
  if (lane == 0) s.warp_top[warp] = top;
  if (tid == 0) s.listed = 0, s.found = -1;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WARPS; ++i) top = fmaxf(top, s.warp_top[i]);
  cluster_wait();
  if (tid < C) cluster.map_shared_rank(s.tops, tid)[rank] = top;
  for (int i = tid; i < kSampleBins; i += kSampleThreads) s.bins[i] = 0;
  cluster.sync();
  for (int i = 0; i < C; ++i) top = fmaxf(top, s.tops[i]);
  // rows that are read again are, where they are aligned, read by runs of four a lane
  const bool runs = !HELD && (reinterpret_cast<uintptr_t>(logits) & (4 * sizeof(T) - 1)) == 0;
  const auto index_of = [&](int j) { return static_cast<uint32_t>(runs ? base + 3 * lane + (j >> 2) * 128 + (j & 3) : base + 32 * j); };
  const bool infinite = top == INFINITY;                                   // infinite logits share the draw
  if constexpr (HELD) {
    if (infinite) {
#pragma unroll 4
      for (int j = 0; j < its; ++j) {
        float& v = s_logits[warp * per_warp + lane + 32 * j];
        v = v == INFINITY ? 0.f : -INFINITY;
      }
    }
  }
  // this lane's j-th of a warp's logits; -inf behind them
  const auto logit_of = [&](int w, int j) {
    if constexpr (HELD) return j < its ? s_logits[w * per_warp + lane + 32 * j] : -INFINITY;
    const int i = rank * a.slice + w * per_warp + lane + 32 * j;
    const float v = j < its && i < a.V ? clean(load_logit(logits + i)) : -INFINITY;
    return !infinite ? v : v == INFINITY ? 0.f : -INFINITY;
  };
  // this lane's logits j0 .. j0 + 3 of its warp's, j0 a multiple of four, as index_of counts them
  const auto fetch = [&](int j0, float (&v)[4]) {
    const int at = static_cast<int>(index_of(j0));
    if (runs && j0 < its && at + 4 <= a.V) {
      T four[4];
      if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(four) = __ldg(reinterpret_cast<const uint4*>(logits + at));
      else *reinterpret_cast<uint2*>(four) = __ldg(reinterpret_cast<const uint2*>(logits + at));
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = to_float(four[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = j0 < its && static_cast<int>(index_of(j0 + i)) < a.V ? load_logit(logits + index_of(j0 + i)) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = clean(v[i]);
      if (infinite) v[i] = v[i] == INFINITY ? 0.f : -INFINITY;
    }
  };
  // f(j, logit) for all of them, N on their way at a time
  const auto for_all = [&](auto n, auto f) {
    constexpr int N = decltype(n)::value;
    if constexpr (HELD) {
#pragma unroll N
      for (int j = 0; j < its; ++j) f(j, s_logits[warp * per_warp + lane + 32 * j]);
    } else {
      for (int j0 = 0; j0 < its; j0 += N) {
        float v[N / 4][4];
#pragma unroll
        for (int i = 0; i < N / 4; ++i) fetch(j0 + 4 * i, v[i]);
#pragma unroll
        for (int i = 0; i < N; ++i) f(j0 + i, v[i >> 2][i & 3]);
      }
    }
  };
  using Four = std::integral_constant<int, 4>;
  using Eight = std::integral_constant<int, 8>;

  // the lowest index of all threads' is the token; none: -1
  const auto write_lowest = [&](uint32_t first) {
    first = __reduce_min_sync(0xffffffffu, first);
    __syncthreads();
    if (lane == 0) s.scan[warp] = first;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < WARPS; ++i) first = min(first, s.scan[i]);
      cluster.map_shared_rank(s.counts, 0)[rank] = first;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
      for (int i = 0; i < C; ++i) first = min(first, s.counts[i]);
      a.token[row] = first == 0xffffffffu ? -1 : static_cast<long long>(first);
    }
  };
  if (top == -INFINITY || !(T_row > 0.0)) {                                // nothing to choose from, or the largest: the lowest index that holds it
    uint32_t first = 0xffffffffu;
    const bool any = top > -INFINITY;
    if (infinite) top = 0.f;                                               // as for_all gives it
    for_all(Eight{}, [&](int j, float v) {
      if (any && v == top) first = min(first, index_of(j));
    });
    write_lowest(first);
    return;
  }
  if (infinite) {
    own_top = own_top == INFINITY ? 0.f : -INFINITY;
    top = 0.f;
  }
  const double c = fmin(fmax(1.4426950408889634 / T_row, 1e-300), 1e300);      // finite: no distance of 0 becomes NaN
  const Weights weigh{exp2(lane / 32.0), static_cast<double>(top), c};
  const double u = a.draws64 ? static_cast<const double*>(a.draws)[row] : static_cast<double>(static_cast<const float*>(a.draws)[row]);
  // A draw of 0 takes the first index that stays and has a weight in 64 bits (2^-1075 and below rounds to none): sums, in which small weights are lost, do not tell it.
  const bool at_start = u <= 0.0;
  const auto weighs = [&](float v) { return (static_cast<double>(v) - weigh.top) * c > -1075.0; };
  const bool by_mass = p < 1.0;
  const float per_bin = fmaxf(fminf(static_cast<float>(c * 64.0), 1e30f), 1e-30f);      // bins of 1/64 of a factor of two; never 0, which no infinite distance takes
  const auto far_of = [&](float v) { return (top - v) * per_bin; };         // in bins; -inf is beyond them all
  const auto bin_of = [&](float v) { return v > -INFINITY ? static_cast<int>(fminf(far_of(v), static_cast<float>(kSampleBins - 1))) : kSampleBins; };

  // the counts of all CTAs' bins, in every CTA
  const auto merge_bins = [&]() {
    cluster.sync();
    const int per = (kSampleBins + C - 1) / C;
    for (int i = rank * per + tid; i < min(kSampleBins, (rank + 1) * per); i += kSampleThreads) {
      uint32_t n = 0;
#pragma unroll
      for (int r = 0; r < kSampleCluster; ++r) n += r < C ? cluster.map_shared_rank(s.bins, r)[i] : 0u;
#pragma unroll
      for (int r = 0; r < kSampleCluster; ++r)
        if (r < C) cluster.map_shared_rank(s.total, r)[i] = n;
    }
    cluster.sync();
  };
  // first bin up to which the merged counts reach `want` (kSampleBins: none); all threads
  const auto bin_reaching = [&](uint32_t want) {
    constexpr int PER = kSampleBins / kSampleThreads;
    uint32_t n[PER], sum = 0, total;
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += n[i] = s.total[tid * PER + i];
    uint32_t upto = block_scan(sum, s.scan, total) - sum;
    if (tid == 0) s.found = kSampleBins;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (upto < want && upto + n[i] >= want) s.found = tid * PER + i;
      upto += n[i];
    }
    __syncthreads();
    return s.found;
  };
  // puts what `take` names into CTA 0's list; its length (beyond the list's end: too many), in every CTA after a cluster.sync()
  const auto gather = [&](auto take) {
    SampleShared* lead = cluster.map_shared_rank(&s, 0);
    for_all(Four{}, [&](int j, float v) {
      const uint32_t key = key_of(v);
      if (key != 0 && take(v, key, index_of(j))) {
        const uint32_t at = atomicAdd(&lead->listed, 1u);
        if (at < kSampleList) lead->list[at] = static_cast<unsigned long long>(key) << 32 | ~index_of(j);
      }
    });
    cluster.sync();
    return lead->listed;
  };
  constexpr int kMaximaK = 128;                                            // with more, too many threads hold several of the k
  constexpr int kFewItems = 256;                                           // 50 items take 0.3 us so and 2.5 by the network, 514 more than by it
  const auto sort_list = [&](int n) {
    if (n <= kFewItems) {
      block_rank(s.list, s.own, n);
      return n;
    }
    int size = 64;
    while (size < n) size <<= 1;
    for (int i = n + tid; i < size; i += kSampleThreads) s.list[i] = 0;
    block_sort(s.list, size);
    return size;
  };

  // whether v lies in bin b, by its distance
  const auto in_bin = [&](float v, float far, int b) { return far >= b && (far < b + 1 || b == kSampleBins - 1) && v > -INFINITY; };

  Place cut{1u, 0xffffffffu};                                              // keeps all

  // ---- top-k -------------------------------------------------------------------------------------------------------------
  if (k_row > 0 && k_row < a.V && k_row <= kSampleList) {
    // the bin with the k-th logit, or with the k-th of the threads' maxima, which lies no higher
    if (k_row <= kMaximaK && a.V >= 64 * k_row) {
      const int own = bin_of(own_top);
      if (own < kSampleBins) atomicAdd(&s.bins[own], 1u);
    } else {
      for_all(Eight{}, [&](int, float v) {
        const int b = bin_of(v);
        if (b < kSampleBins) atomicAdd(&s.bins[b], 1u);
      });
    }
    merge_bins();
    const int last = bin_reaching(k_row);                                  // none: not that many
    if (tid == 0) s.collected = 0;
    __syncthreads();
    if (last < kSampleBins - 1) {
      for_all(Eight{}, [&](int j, float v) {
        if (far_of(v) < last + 1) {
          const uint32_t at = atomicAdd(&s.collected, 1u);
          if (at < kSampleList) s.own[at] = static_cast<unsigned long long>(key_of(v)) << 32 | ~index_of(j);
        }
      });
    }
    __syncthreads();
    const uint32_t own_n = s.collected;
    if (tid < C) cluster.map_shared_rank(s.counts, tid)[rank] = own_n;
    cluster.sync();                                                        // from here on nobody looks at logits, if all fits
    uint32_t before = 0, n = 0;
    bool fits = last < kSampleBins - 1;
    for (int r = 0; r < C; ++r) {
      fits &= s.counts[r] <= kSampleList;
      if (r < rank) before += s.counts[r];
      n += s.counts[r];
    }
    fits &= n <= kSampleMost;
    if (fits) {
      unsigned long long* list = reinterpret_cast<unsigned long long*>(s_logits);
      unsigned long long* to = cluster.map_shared_rank(list, 0) + before;
      for (int i = tid; i < static_cast<int>(own_n); i += kSampleThreads) to[i] = s.own[i];
      cluster.sync();
      if (rank != 0) return;
      // ---- all that can stay lies in CTA 0's list: weights as whole numbers of 2^-52, whose sums do not depend on their order -----------
      unsigned long long *some = list + kSampleMost, *some_w = some + kSampleMost;
      constexpr int PER = kSampleMost / kSampleThreads, BINS = kSampleBins / kSampleThreads;
      constexpr double kUnit = 4503599627370496.0;
      // the first index whose running weight passes the aim, else the last: from the items (~index in their lower halves), their weights and what lies before them
      const auto draw_from = [&](unsigned long long item, unsigned long long w, unsigned long long base, const unsigned long long* items, const unsigned long long* weights, int n,
                                 double aim) {
        if (w == 0) return;
        const uint32_t mine = static_cast<uint32_t>(item);
        unsigned long long upto = base;
        for (int j = 0; j < n; ++j) upto += static_cast<uint32_t>(items[j]) >= mine ? weights[j] : 0ull;
        if (static_cast<double>(upto) > aim) atomicMax(&s.best, static_cast<unsigned long long>(mine) + 1);
        atomicMax(&s.bests[0], static_cast<unsigned long long>(~mine) + 1);
      };
      const auto write_token = [&]() {
        __syncthreads();
        if (tid == 0) a.token[row] = s.best != 0 ? ~static_cast<uint32_t>(s.best - 1) : static_cast<uint32_t>(s.bests[0] - 1);
      };
      if (n <= kFewItems) {                                                // one a thread, in order: 50 items take 7 us less so than by bins
        block_rank(list, some, n);
        const unsigned long long mine = tid < static_cast<int>(n) ? list[tid] : 0;
        bool stay = tid < min(static_cast<int>(n), k_row);
        const double exact = weigh(stay ? value_of(static_cast<uint32_t>(mine >> 32)) : top);
        unsigned long long w = stay ? static_cast<unsigned long long>(exact * kUnit) : 0, total;
        const unsigned long long ahead = block_scan_u(w, s.scan_u, total) - w;
        stay &= exact >= m && (!by_mass || tid == 0 || static_cast<double>(ahead) < p * static_cast<double>(total));
        if (!stay) w = 0;
        if (tid < static_cast<int>(n)) some_w[tid] = w;
        if (tid == 0) s.best = 0, s.bests[0] = 0;
        block_scan_u(w, s.scan_u, total);
        if (!at_start) draw_from(mine, w, 0, list, some_w, n, u * static_cast<double>(total));
        else if (stay && weighs(value_of(static_cast<uint32_t>(mine >> 32)))) atomicMax(&s.best, static_cast<unsigned long long>(static_cast<uint32_t>(mine)) + 1);
        write_token();
        return;
      }
      unsigned long long item[PER], w[PER];
      int bin[PER];
      bool in[PER];
      for (int i = tid; i < kSampleBins; i += kSampleThreads) s.total[i] = 0;
      __syncthreads();
#pragma unroll
      for (int r = 0; r < PER; ++r) {
        const int i = tid + r * kSampleThreads;
        in[r] = i < static_cast<int>(n);
        item[r] = in[r] ? list[i] : 0;
        const float v = in[r] ? value_of(static_cast<uint32_t>(item[r] >> 32)) : top;
        w[r] = static_cast<unsigned long long>(weigh(v) * kUnit);
        bin[r] = bin_of(v);
        if (in[r]) atomicAdd(&s.total[bin[r]], 1u);
      }
      __syncthreads();
      // items of one bin, listed in any order: their number, after a barrier
      const auto bring = [&](int b, const int (&of)[PER]) {
        __syncthreads();
        if (tid == 0) s.collected = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < PER; ++r)
          if (in[r] && of[r] == b) {
            const uint32_t at = atomicAdd(&s.collected, 1u);
            some[at] = item[r];
            some_w[at] = w[r];
          }
        __syncthreads();
        return static_cast<int>(s.collected);
      };
      const int cut_k = bin_reaching(min(static_cast<uint32_t>(k_row), n));
      uint32_t above = 0, all;
      for (int i = tid; i < cut_k; i += kSampleThreads) above += s.total[i];
      block_scan(above, s.scan, all);
      const int some_n = bring(cut_k, bin);
#pragma unroll
      for (int r = 0; r < PER; ++r) {
        if (in[r] && bin[r] == cut_k) {
          int rank_in = 0;
          for (int j = 0; j < some_n; ++j) rank_in += some[j] > item[r];
          in[r] = rank_in < k_row - static_cast<int>(all);
        } else {
          in[r] &= bin[r] < cut_k;
        }
      }
      // weights by bins (any numbering of 2048), and the bin in which their running sum passes `aim`, with what lies before it; the last that holds any, else
      const auto passing_bin = [&](const int (&of)[PER], auto passes) {
        __syncthreads();
        for (int i = tid; i < kSampleBins; i += kSampleThreads) s.mass[i] = 0;
        if (tid == 0) s.found = kSampleBins, s.flag = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < PER; ++r)
          if (in[r] && w[r] != 0) atomicAdd(&s.mass[of[r]], w[r]);
        __syncthreads();
        unsigned long long sum = 0, total, v[BINS];
#pragma unroll
        for (int i = 0; i < BINS; ++i) sum += v[i] = s.mass[tid * BINS + i];
        unsigned long long upto = block_scan_u(sum, s.scan_u, total) - sum, start[BINS];
        passes(0ull, total);                                               // every thread learns the whole
#pragma unroll
        for (int i = 0; i < BINS; ++i) {
          start[i] = upto;
          upto += v[i];
          if (v[i] == 0) continue;
          atomicMax(&s.flag, tid * BINS + i);
          if (passes(upto, total)) atomicMin(&s.found, tid * BINS + i);
        }
        __syncthreads();
        const int at = s.found < kSampleBins ? s.found : s.flag;
#pragma unroll
        for (int i = 0; i < BINS; ++i)
          if (tid * BINS + i == at) s.base = start[i];
        __syncthreads();
        return at;
      };
      if (by_mass) {
        unsigned long long whole = 0, total;
#pragma unroll
        for (int r = 0; r < PER; ++r) whole += in[r] ? w[r] : 0;
        block_scan_u(whole, s.scan_u, total);
        const double aim = fmax(p * static_cast<double>(total), 0.5);       // nothing lies before the first
        const int at = passing_bin(bin, [&](unsigned long long upto, unsigned long long) { return static_cast<double>(upto) >= aim; });
        const unsigned long long base = s.base;
        const int m_n = bring(at, bin);
#pragma unroll
        for (int r = 0; r < PER; ++r) {
          if (in[r] && bin[r] == at) {
            unsigned long long ahead = base;
            for (int j = 0; j < m_n; ++j) ahead += some[j] > item[r] ? some_w[j] : 0ull;
            in[r] = static_cast<double>(ahead) < aim;
          } else {
            in[r] &= bin[r] < at;
          }
        }
      }
      // the draw, in vocabulary order
#pragma unroll
      for (int r = 0; r < PER; ++r) {
        const double exact = weigh(in[r] ? value_of(static_cast<uint32_t>(item[r] >> 32)) : top);
        in[r] = in[r] && exact >= m;
        bin[r] = static_cast<int>(static_cast<unsigned long long>(~static_cast<uint32_t>(item[r])) * kSampleBins / static_cast<unsigned>(a.V));
      }
      if (at_start) {
        if (tid == 0) s.best = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < PER; ++r)
          if (in[r] && weighs(value_of(static_cast<uint32_t>(item[r] >> 32)))) atomicMax(&s.best, static_cast<unsigned long long>(static_cast<uint32_t>(item[r])) + 1);
        write_token();
        return;
      }
      double draw_aim = 0.0;
      const int at = passing_bin(bin, [&](unsigned long long upto, unsigned long long total) {
        draw_aim = u * static_cast<double>(total);
        return static_cast<double>(upto) > draw_aim;
      });
      const unsigned long long base = s.base;
      if (tid == 0) s.best = 0, s.bests[0] = 0;
      const int d_n = bring(at, bin);
#pragma unroll
      for (int r = 0; r < PER; ++r)
        if (in[r] && bin[r] == at) draw_from(item[r], w[r], base, some, some_w, d_n, draw_aim);
      write_token();
      return;
    }
    for (int i = tid; i < kSampleBins; i += kSampleThreads) s.bins[i] = 0;
    if (tid == 0) s.listed = 0;
    cluster.sync();
  }

  const auto fix_of = [&](float largest) {                                 // 2^52 over the power of two above its weight
    return __hiloint2double((2046 + 52 - (__double2hiint(weigh(largest)) >> 20 & 0x7ff)) << 20, 0);
  };
  float cut_high = 0.f;
  // One cut in the order: by the number of what stays (k), or by its weight (below p times the weight of all that the present cut keeps).
  int cut_bin = -1;                                                        // the bin of values in which a cut by weight over all lies
  const auto select = [&](bool mass, uint32_t k) __attribute__((always_inline)) {
    const bool whole = cut.key == 1u;                                      // nothing is cut yet
    uint32_t low = 0, high = 0xffffffffu, above_n = 0;
    double above = 0.0, aim = 0.0;
    bool first = true;
    int shift = 0, turn = mass;
    uint32_t in_n;
    int last_turn = 0;
    // bins of the present interval: by value over all, then by key
    const auto place = [&](float v, uint32_t key) { return first ? bin_of(v) : static_cast<int>((high - key) >> shift); };
    const auto inside = [&](uint32_t key, uint32_t index) { return key != 0 && key >= low && key <= high && stays(key, index, cut); };
    do {                                                                   // by value, then 2^32 keys by 2048 bins three times at most
      if (first && whole) {
        for_all(Eight{}, [&](int, float v) {
          const int b = bin_of(v);
          if (b < kSampleBins) atomicAdd(&s.bins[b], 1u);
        });
      } else {
        for_all(Four{}, [&](int j, float v) {
          const uint32_t key = key_of(v);
          if (inside(key, index_of(j))) atomicAdd(&s.bins[place(v, key)], 1u);
        });
      }
      merge_bins();
      for (int i = tid; i < kSampleBins; i += kSampleThreads) s.bins[i] = 0;
      int bin;
      Partial all;
      // weights above, in and below a bin of the interval
      const auto weigh_bin = [&](int b) {
        Partial q{0.0, 0.0, 0.0, 0u, 0xffffffffu, 0u, 0u};            // `all` counts only over the first interval
        const auto note = [&](uint32_t key) {
          ++q.count;
          q.low = min(q.low, key);
          q.high = max(q.high, key);
        };
        if (mass && first && whole) {
          if (tid == 0) s.collected = 0;
          __syncthreads();
          float ahead[4];
          if constexpr (!HELD) fetch(0, ahead);
          for (int j0 = 0; j0 < its; j0 += 4) {                            // four weights hide each other's latency
            float v[4];
            double w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = HELD ? logit_of(warp, j0 + i) : ahead[i];
            if constexpr (!HELD) fetch(j0 + 4, ahead);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = weigh(v[i]);
            bool hit[4], any = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float far = far_of(v[i]);
              q.all += w[i];
              if (far < b) q.above += w[i];
              any |= hit[i] = in_bin(v[i], far, b);
            }
            if (any) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (!hit[i]) continue;
                const uint32_t key = key_of(v[i]);
                q.in += w[i];
                note(key);
                const uint32_t at = atomicAdd(&s.collected, 1u);
                if (at < kSampleList) s.own[at] = static_cast<unsigned long long>(key) << 32 | ~index_of(j0 + i);
              }
            }
          }
        } else {
          for_all(Four{}, [&](int j, float v) {
            const uint32_t key = key_of(v);
            const bool is_in = inside(key, index_of(j));
            const int at = is_in ? place(v, key) : 0;
            if (mass && __any_sync(0xffffffffu, is_in)) {
              const double w = weigh(v);
              if (is_in) {
                q.all += w;
                if (at <= b) (at < b ? q.above : q.in) += w;
              }
            }
            if (is_in && at == b) note(key);
          });
        }
        q.above = warp_sum_d(q.above), q.in = warp_sum_d(q.in), q.all = warp_sum_d(q.all);
        if (lane == 0) s.warp_above[warp] = q.above;
        q.count = __reduce_add_sync(0xffffffffu, q.count);
        q.low = __reduce_min_sync(0xffffffffu, q.low);
        q.high = __reduce_max_sync(0xffffffffu, q.high);
        const auto join = [](Partial& x, const Partial& y) {
          x.above += y.above, x.in += y.in, x.all += y.all, x.count += y.count;
          x.low = min(x.low, y.low), x.high = max(x.high, y.high);
        };
        if (lane == 0) s.warp_part[warp] = q;
        __syncthreads();
        q = s.warp_part[0];
#pragma unroll
        for (int i = 1; i < WARPS; ++i) join(q, s.warp_part[i]);
        turn ^= 1;
        if (tid < C) cluster.map_shared_rank(s.part[turn], tid)[rank] = q;
        cluster.sync();                                                    // behind it nobody reads the parts of the call before the last
        q = s.part[turn][0];
        for (int i = 1; i < C; ++i) join(q, s.part[turn][i]);
        return q;
      };
      if (!mass) {
        bin = bin_reaching(k - above_n);
        if (bin == kSampleBins) return;                                    // no more than k to choose from
        all = weigh_bin(bin);
        // what lies above the bin, from the counts
        uint32_t n = 0, total;
        for (int i = tid; i < bin; i += kSampleThreads) n += s.total[i];
        block_scan(n, s.scan, total);
        above_n += total;
      } else {
        // where the counts, each taken at its bin's middle, reach the aim; exact sums then say how far off that is
        constexpr int PER = kSampleBins / kSampleThreads;
        double est[PER], sum = 0.0, total;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int b = tid * PER + i;
          const double mid = first ? static_cast<double>(top) - (b + 0.5) / static_cast<double>(per_bin)
                                   : static_cast<double>(value_of(max(low, high - min(high - low, (static_cast<uint32_t>(b) << shift) + ((1u << shift) >> 1)))));
          est[i] = s.total[b] * static_cast<double>(exp2f(static_cast<float>(fmax((mid - static_cast<double>(top)) * c, -140.0))));
          sum += est[i];
        }
        const double est_before = block_scan_d(sum, s.scan_d, total) - sum;
        double want = first ? p * total : aim - above;
        int least = 0, most = kSampleBins - 1;
        bool again;
        do {                                                               // each time leaves a bin out
          if (tid == 0) s.found = kSampleBins, s.flag = least;
          __syncthreads();
          double upto = est_before;
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const int b = tid * PER + i;
            upto += est[i];
            if (s.total[b] && b >= least && b <= most) {
              if (upto >= want) atomicMin(&s.found, b);
              atomicMax(&s.flag, b);                                       // the last that holds any
            }
          }
          __syncthreads();
          bin = min(s.found, s.flag);
          // the estimate of what lies above it
          if (tid == bin / PER) {
            double e = est_before;
#pragma unroll
            for (int i = 0; i < PER; ++i)
              if (tid * PER + i < bin) e += est[i];
            s.scan_d[0] = e;
          }
          __syncthreads();
          const double est_above = s.scan_d[0];
          all = weigh_bin(bin);
          if (first) aim = fmax(p * all.all, 1e-300);
          const double goal = aim - above;
          again = true;
          if (goal <= all.above && bin > least) most = bin - 1;             // the cut lies further up ...
          else if (goal > all.above + all.in && bin < most) least = bin + 1;     // ... or down
          else again = false;
          want = goal + (est_above - all.above);
        } while (again);
        above += all.above;
      }
      in_n = all.count;
      last_turn = turn;
      low = all.low;
      high = all.high;
      if (low < high && in_n > kSampleList) {
        first = false;
        shift = 0;
        while (((high - low) >> shift) >= static_cast<uint32_t>(kSampleBins)) ++shift;
      } else if (mass && first && whole && in_n <= kSampleList) {
        cut_bin = bin, cut_high = value_of(high);
      }
    } while (low < high && in_n > kSampleList);
    const auto member = [&](uint32_t key, uint32_t index) { return key >= low && key <= high && stays(key, index, cut); };
    if (in_n <= kSampleList) {
      if (mass && first && whole) {
        // collected beside the sums: every CTA gets all of it and places its own, by the weight of what comes before.  Weights here are whole numbers, of the
        // largest's 2^-52, so that their sums do not depend on the order in which they were collected.
        const int own_n = s.part[last_turn][rank].count;
        uint32_t before = 0;
        for (int r = 0; r < rank; ++r) before += s.part[last_turn][r].count;
        for (int i = tid; i < own_n * C; i += kSampleThreads) cluster.map_shared_rank(&s, i / own_n)->list[before + i % own_n] = s.own[i % own_n];
        if (tid == 0) s.best = ~0ull;
        cluster.sync();
        const double unit = fix_of(value_of(high));
        for (int i = tid; i < (static_cast<int>(in_n) + 31) / 32 * 32; i += kSampleThreads) {      // whole warps weigh
          const double w = weigh(value_of(static_cast<uint32_t>(s.list[min(i, static_cast<int>(in_n) - 1)] >> 32)));
          if (i < static_cast<int>(in_n)) s.fixed[i] = static_cast<unsigned long long>(w * unit);
        }
        __syncthreads();
        const int each = own_n > 256 ? 1 : own_n > 128 ? 2 : own_n > 64 ? 4 : own_n > 32 ? 8 : own_n > 16 ? 16 : 32;      // threads an item
        for (int i0 = 0; i0 < own_n; i0 += kSampleThreads / each) {
          const int i = i0 + tid / each;
          const unsigned long long item = s.own[min(i, own_n - 1)];
          unsigned long long ahead = 0;
          for (int j = tid % each; j < static_cast<int>(in_n); j += each) ahead += s.list[j] > item ? s.fixed[j] : 0ull;
          for (int o = 1; o < each; o <<= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
          if (i < own_n && tid % each == 0 && above + static_cast<double>(ahead) / unit < aim) atomicMin(&s.best, item);
        }
        __syncthreads();
        if (tid < C) cluster.map_shared_rank(s.bests, tid)[rank] = s.best;
        cluster.sync();
        unsigned long long last = ~0ull;
        for (int r = 0; r < C; ++r) last = min(last, s.bests[r]);
        if (last == ~0ull) last = static_cast<unsigned long long>(high) << 32;      // not even the first: by a rounding of the sums alone
        cut = Place{static_cast<uint32_t>(last >> 32), ~static_cast<uint32_t>(last)};
        return;
      }
      const uint32_t n = gather([&](float, uint32_t key, uint32_t index) { return member(key, index); });
      if (rank == 0) {
        sort_list(n);
        int last;                                                          // the last of the list that stays
        if (!mass) {
          last = static_cast<int>(k - above_n) - 1;
        } else {
          constexpr int PER = kSampleList / kSampleThreads;
          double w[PER], sum = 0.0, total;
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const int at = tid * PER + i;
            const double v = weigh(at < static_cast<int>(n) ? value_of(static_cast<uint32_t>(s.list[at] >> 32)) : 0.f);
            w[i] = at < static_cast<int>(n) ? v : 0.0;
            sum += w[i];
          }
          double before = above + block_scan_d(sum, s.scan_d, total) - sum;
          if (tid == 0) s.flag = 0;
          __syncthreads();
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            if (tid * PER + i < static_cast<int>(n) && before < aim) atomicMax(&s.flag, tid * PER + i);
            before += w[i];
          }
          __syncthreads();
          last = s.flag;
        }
        if (tid < C) {
          const unsigned long long it = s.list[last];
          cluster.map_shared_rank(&s, tid)->cut = Place{static_cast<uint32_t>(it >> 32), ~static_cast<uint32_t>(it)};
        }
      }
    } else {
      // more equal logits than the list holds: the first ones in vocabulary order
      double w = weigh(value_of(high));
      const double take = mass ? ceil((aim - above) / w) : static_cast<double>(k - above_n);
      const uint32_t want = take >= in_n ? in_n : take < 1.0 ? 1u : static_cast<uint32_t>(take);
      uint32_t n = 0;
      for_all(Four{}, [&](int j, float v) { n += member(key_of(v), index_of(j)) ? 1u : 0u; });
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane < C) cluster.map_shared_rank(s.counts, lane)[rank * WARPS + warp] = n;
      cluster.sync();
      uint32_t before = 0;
      for (int i = lane; i < rank * WARPS + warp; i += 32) before += s.counts[i];
      before = __reduce_add_sync(0xffffffffu, before);
      if (before < want && before + n >= want) {
#pragma unroll 4
        for (int j = 0; j < its; ++j) {                                    // in vocabulary order
          const uint32_t index = base + 32 * j, in = __ballot_sync(0xffffffffu, member(key_of(logit_of(warp, j)), index));
          const uint32_t mine = before + __popc(in & ((2u << lane) - 1u));
          if (before < want && before + __popc(in) >= want && (in >> lane & 1) && mine == want)
            for (int r = 0; r < C; ++r) cluster.map_shared_rank(&s, r)->cut = Place{high, index};
          before += __popc(in);
        }
      }
    }
    cluster.sync();
    cut = s.cut;
    if (!mass) {                                                           // the list may be wanted once more
      if (tid == 0) s.listed = 0;
      cluster.sync();
    }
  };
  if (k_row > 0 && k_row < a.V) select(false, k_row);
  if (by_mass) select(true, 0);

  // ---- the draw ------------------------------------------------------------------------------------------------------------
  if (at_start) {
    uint32_t first = 0xffffffffu;
    for_all(Four{}, [&](int j, float v) {
      const uint32_t key = key_of(v);
      const bool heavy = m <= 0.0 || weigh(v) >= m;
      if (key != 0 && heavy && weighs(v) && stays(key, index_of(j), cut)) first = min(first, index_of(j));
    });
    write_lowest(first);
    return;
  }
  const float low_m = m > 0.0 ? static_cast<float>(top + log2(m) / c - 1e-6 * (fabs(top) + fabs(log2(m) / c))) : -INFINITY;      // no weight below it reaches min_p
  const auto weight_of = [&](int j, float v) {
    const uint32_t key = key_of(v);
    const bool in = key != 0 && v >= low_m && stays(key, index_of(j), cut);
    if (!__any_sync(0xffffffffu, in)) return 0.0;
    const double w = weigh(v);
    return in && w >= m ? w : 0.0;
  };
  double sum = 0.0;
  if (cut.key == 1u && m <= 0.0) {
    for_all(std::integral_constant<int, HELD ? 4 : 8>{}, [&](int, float v) { sum += weigh(v); });
    sum = warp_sum_d(sum);
    if (sum < 1e-200) sum = 0.0;                                           // nothing but what is never chosen
  } else if (cut_bin >= 0 && m <= 0.0) {
    // what lies above the cut's bin has been summed up, and what lies in it is listed
    if (tid < WARPS) s.fixed[tid] = 0;
    __syncthreads();
    const double unit = fix_of(cut_high);
    const int own_n = s.collected;
    for (int i = tid; i < (own_n + 31) / 32 * 32; i += kSampleThreads) {
      const unsigned long long item = s.own[min(i, own_n - 1)];
      const uint32_t key = static_cast<uint32_t>(item >> 32), index = ~static_cast<uint32_t>(item);
      const double w = weigh(value_of(key));
      if (i < own_n && stays(key, index, cut)) atomicAdd(&s.fixed[(index - rank * a.slice) / per_warp], static_cast<unsigned long long>(w * unit));
    }
    __syncthreads();
    sum = s.warp_above[warp] + static_cast<double>(s.fixed[warp]) / unit;
  } else {
    for_all(Four{}, [&](int j, float v) { sum += weight_of(j, v); });
    sum = warp_sum_d(sum);
  }
  // the CTA in which the cumulative weight passes the aim, else the last that holds any; then the warp in it, then the run of 32
  if (lane == 0) s.warp_sums[warp] = sum;
  __syncthreads();
  if (tid < C) {
    double own = 0.0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) own += s.warp_sums[i];
    cluster.map_shared_rank(s.cta_sums, tid)[rank] = own;
  }
  cluster.sync();
  // (which of the lanes' numbers in a row passes the aim, what lies before it); the last that holds any where none does
  const auto passing = [&](double v, double start, double aim, double& before) {
    const double upto = start + warp_scan_d(v, lane);
    const uint32_t any = __ballot_sync(0xffffffffu, v > 0.0), past = __ballot_sync(0xffffffffu, v > 0.0 && upto > aim);
    const int at = past ? __ffs(past) - 1 : 31 - __clz(any | 1u);
    before = __shfl_sync(0xffffffffu, upto - v, at);
    return at;
  };
  const double cta = lane < C ? s.cta_sums[lane] : 0.0, aim = u * warp_sum_d(cta);
  double before;
  if (passing(cta, 0.0, aim, before) != rank) return;
  const int at_warp = passing(lane < WARPS ? s.warp_sums[lane] : 0.0, before, aim, before);
  // all warps weigh that warp's logits, each its runs
  const uint32_t part_index = rank * a.slice + at_warp * per_warp + lane;
  const auto weight_at = [&](int j) {
    const float v = logit_of(at_warp, j);
    const uint32_t key = key_of(v);
    const double w = weigh(v);
    return key != 0 && stays(key, part_index + 32 * j, cut) && w >= m ? w : 0.0;
  };
  for (int j = warp; j < its; j += WARPS) {
    const double run = warp_sum_d(weight_at(j));
    if (lane == 0) s.run_sums[j] = run;
  }
  __syncthreads();
  if (warp != 0) return;
  int at_run = -1, last_run = 0;
  double last_before = before;
  for (int j0 = 0; j0 < its && at_run < 0; j0 += 32) {
    const double v = j0 + lane < its ? s.run_sums[j0 + lane] : 0.0;
    const double upto = before + warp_scan_d(v, lane);
    const uint32_t any = __ballot_sync(0xffffffffu, v > 0.0), past = __ballot_sync(0xffffffffu, v > 0.0 && upto > aim);
    if (any) {
      const int at = past ? __ffs(past) - 1 : 31 - __clz(any);
      last_run = j0 + at;
      last_before = __shfl_sync(0xffffffffu, upto - v, at);
      if (past) at_run = last_run;
    }
    before = __shfl_sync(0xffffffffu, upto, 31);
  }
  double unused;
  const int at = passing(weight_at(last_run), last_before, aim, unused);
  if (lane == at) a.token[row] = part_index + 32 * last_run;
}

template <typename T, bool HELD>
int sample_form(const SampleArgs& a, int ctas, cudaStream_t stream) {
  static OncePerDevice ready;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -4;
  const int failed = ready(dev, [] {
    const cudaError_t e = cudaFuncSetAttribute(sample_kernel<T, HELD>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    return static_cast<int>(e != cudaSuccess ? e : cudaFuncSetAttribute(sample_kernel<T, HELD>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSampleLargest * 4));
  });
  if (failed != 0) return failed;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows) * ctas);
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = HELD && a.slice * 4 > kSampleScratch ? a.slice * 4 : kSampleScratch;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, sample_kernel<T, HELD>, a));
}

template <typename T>
int sample_any(SampleArgs a, cudaStream_t stream) {
  // the fewest CTAs a row that leave room for two on an SM; more while there are few rows
  int ctas = 1;
  while (ctas < kSampleCluster && (static_cast<long long>(ctas) * kSampleSlice < a.V || (a.rows * ctas * 2 <= 148 && ctas * kSampleThreads * 4 < a.V))) ctas *= 2;
  if (static_cast<long long>(ctas) * kSampleLargest < a.V) return -2;
  const int held = ctas;
  // Where that would take three rounds and more, fewer CTAs a row that read it anew for every pass: fewer steps in which they wait for one another.  In us, held /
  // read, fp32: 128 x 262144 by top-p 401 / 262, by top-k 133 / 74, no filter 120 / 91; 256 x 50304 157 / 93, 70 / 33, 50 / 37.  With less it depends: 48 x 248320 in
  // bf16, 2.6 rounds, by top-p 152 / 125, no filter 42 / 50, settings of all kinds 88 / 116, since a row that is cut by mass holds up all.
  if (static_cast<long long>(a.rows) * ctas > 3 * 296)
    while (ctas > 1 && static_cast<long long>(a.rows) * ctas > 296 && static_cast<long long>(ctas / 2) * kSampleRead >= a.V) ctas /= 2;
  const int step = ctas * kSampleThreads * (ctas == held ? 1 : 4);          // whole runs of four where rows are read again
  a.slice = (a.V + step - 1) / step * step / ctas;
  return ctas == held ? sample_form<T, true>(a, ctas, stream) : sample_form<T, false>(a, ctas, stream);
}

}  // namespace tyr

using namespace tyr;

// dtype: 0 = bf16, 1 = fp16, 2 = fp32 (the logits)
extern "C" TYR_EXPORT int tyr_sample(const void* packed, int dtype, void* stream) {
  const SampleArgs& a = *static_cast<const SampleArgs*>(packed);
  if (a.rows <= 0 || a.V <= 0 || a.rows > (1 << 26)) return -1;
  switch (dtype) {
    case 0: return sample_any<__nv_bfloat16>(a, (cudaStream_t)stream);
    case 1: return sample_any<__half>(a, (cudaStream_t)stream);
    case 2: return sample_any<float>(a, (cudaStream_t)stream);
  }
  return -3;
}
