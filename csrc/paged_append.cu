// Keys and values of new tokens into a paged cache, with the per-head RMS norm and the rotation by position on the way, and the queries with them.
//
// Pages [pages, G, P, D] hold P tokens of G heads, in 16 bits or as e4m3 codes in units of a scale for each (page, head): scale 2^e with the smallest
// e >= -100 that keeps the page's largest magnitude within 448.  A page that was begun by an earlier call keeps its scale while the new tokens fit, else the
// larger one replaces it and the older codes are rescaled; by a power of two that is exact unless they leave e4m3's normal range.  A value that is not finite
// makes the scale NaN, so that what attends the page shows it.
//
// Row r of sequence b is at position lengths[b] - n + (r - starts[b]) with n = starts[b + 1] - starts[b] (no starts: one row each, n = 1 where the length is
// at least 1).  Compiled without fast math.
//
// Bound: memory for many rows, each of which is read once and written once.  8 x 4096 tokens, 48 query and 8 K/V heads of 128, bf16 into e4m3: 185 us, 4.9 TB/s; 9 x some
// 300 tokens, 24 and 4 heads of 256, fp16 pages: 26.5 us, 2.9 TB/s.  Registers bound the copies in flight; loading rows before their sequence or page is
// looked up took the second to 25.9 us and the first to 191, by spills.
#include <cuda_fp8.h>

#include "common.cuh"

namespace tyr {

struct PagedAppendArgs {
  const void *q, *k, *v;                    // [rows, heads, D]; element strides of rows and heads below
  void* q_out;                              // [rows, H, D]
  void *k_pages, *v_pages;                  // [pages, G, P, D]
  float *k_scale, *v_scale;                 // [pages, G] (null: 16-bit pages)
  const int *table, *lengths, *starts;      // [B, width], [B], [B + 1] (nullable)
  const float *cos, *sin;                   // [positions, half] (null: no rotation)
  const void *q_weight, *k_weight;          // [D] (nullable)
  int* err;
  long long q_row, q_head, k_row, k_head, v_row, v_head, table_row;
  int rows, B, H, G, D, P, pages, width, positions, half, one_plus_w;
  float eps;
};
static_assert(sizeof(PagedAppendArgs) == 232, "as ops/paged_cache.py packs it");

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ float2 get(uint32_t u) { return unpack_bf16x2(u); }
  static __device__ __forceinline__ uint32_t put(float a, float b) { return pack_bf16x2(a, b); }
};
template <> struct Pair<__half> {
  static __device__ __forceinline__ float2 get(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
  static __device__ __forceinline__ uint32_t put(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// Eight channels of a lane are two runs of four: `raw` holds them as they lie in memory.
template <typename T>
__device__ __forceinline__ void pa_unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = Pair<T>::get(w[i]);
    f[2 * i] = t.x; f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ uint2 pa_codes8(const float (&f)[8], float inv) {      // zeros for a scale that is NaN (inv 0): codes are numbers always
  if (inv == 0.f) return make_uint2(0u, 0u);
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i] * inv, f[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
}
__device__ __forceinline__ uint32_t pa_recode4(uint32_t codes, float ratio) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes >> 16 * i), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    out |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(f.x * ratio, f.y * ratio), __NV_SATFINITE, __NV_E4M3)) << 16 * i;
  }
  return out;
}

__device__ __forceinline__ uint32_t pa_magnitude(const float (&f)[8]) {      // the bits of magnitudes order like the magnitudes, infinities and NaN above all
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  return m;
}
// The scale of a page whose largest magnitude has these bits.
__device__ __forceinline__ float pa_scale(uint32_t bits) {
  if (bits >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
  const int e = static_cast<int>(bits >> 23) - 135 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);      // 448 = 1.75 * 2^8
  return __uint_as_float(static_cast<uint32_t>(max(e, -100) + 127) << 23);
}
// ... of one that also holds older tokens in units of `old`
__device__ __forceinline__ float pa_joined(float want, float old) { return want != want || old != old ? __uint_as_float(0x7fffffffu) : fmaxf(want, old); }
__device__ __forceinline__ float pa_inverse(float scale) { return scale == scale ? 1.f / scale : 0.f; }

// A head on D / 8 neighbouring lanes, all of whose rows are at one position.  Of the rotated part a lane has four channels and the four that they turn with, so that
// the rotation needs no other lane; of the rest eight in a row.
struct HeadLanes {
  int lane, lanes, lo, hi;                     // channels lo .. lo + 3 and hi .. hi + 3
  bool turned;
  uint32_t mask;
  float4 c, s;
  __device__ __forceinline__ HeadLanes(const PagedAppendArgs& a, int thread)
      : lanes(a.D >> 3), mask(a.D == 256 ? 0xffffffffu : ((1u << (a.D >> 3)) - 1u) << ((threadIdx.x & 31) & ~((a.D >> 3) - 1))) {
    lane = thread & (lanes - 1);
    const int pairs = a.half >> 2;
    turned = lane < pairs;
    lo = turned ? 4 * lane : 2 * a.half + 8 * (lane - pairs);
    hi = turned ? a.half + lo : lo + 4;
  }
  template <typename T>
  __device__ __forceinline__ uint4 raw(const T* head) const {
    const uint2 x = *reinterpret_cast<const uint2*>(head + lo), y = *reinterpret_cast<const uint2*>(head + hi);
    return make_uint4(x.x, x.y, y.x, y.y);
  }
  template <typename T>
  __device__ __forceinline__ void store(T* head, const float (&f)[8]) const {
    *reinterpret_cast<uint2*>(head + lo) = make_uint2(Pair<T>::put(f[0], f[1]), Pair<T>::put(f[2], f[3]));
    *reinterpret_cast<uint2*>(head + hi) = make_uint2(Pair<T>::put(f[4], f[5]), Pair<T>::put(f[6], f[7]));
  }
  __device__ __forceinline__ void store_codes(uint8_t* head, const float (&f)[8], float inv) const {
    const uint2 u = pa_codes8(f, inv);
    *reinterpret_cast<uint32_t*>(head + lo) = u.x;
    *reinterpret_cast<uint32_t*>(head + hi) = u.y;
  }
  __device__ __forceinline__ void turns(const PagedAppendArgs& a, int pos) {
    if (!turned) return;
    const long long at = static_cast<long long>(pos) * a.half + lo;
    c = *reinterpret_cast<const float4*>(a.cos + at);
    s = *reinterpret_cast<const float4*>(a.sin + at);
  }
  // norm and rotation of the lanes' channels, in 32 bits throughout
  template <typename T>
  __device__ __forceinline__ void finish(const PagedAppendArgs& a, const T* weight, float (&f)[8]) const {
    if (weight != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
      for (int o = lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
      const float r = rsqrtf(ss / a.D + a.eps);
      float w[8];
      pa_unpack8<T>(raw(weight), w);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = f[i] * r * (a.one_plus_w ? 1.f + w[i] : w[i]);
    }
    if (turned) {
      const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = f[i], y = f[4 + i];
        f[i] = x * cs[i] - y * sn[i];
        f[4 + i] = x * sn[i] + y * cs[i];
      }
    }
  }
};

// What sequence b brings: first row, rows and the position of the first; no rows where the operands do not go together (recorded).
struct NewRows { int row, n, first; };
__device__ __forceinline__ NewRows pa_new_rows(const PagedAppendArgs& a, int b) {
  const int len = a.lengths[b];
  const int row = a.starts ? a.starts[b] : b, n = a.starts ? a.starts[b + 1] - row : (len > 0 ? 1 : 0);
  if (n == 0) return {row, 0, len};
  if (n < 0 || row < 0 || row + n > a.rows || len < n || (len - 1) / a.P >= a.width || (a.half > 0 && len > a.positions)) {
    report_error(a.err, ERR_BOUNDS, b);
    return {row, 0, len};
  }
  return {row, n, len - n};
}
__device__ __forceinline__ int pa_page(const PagedAppendArgs& a, int b, int j) {
  const int page = a.table[b * a.table_row + j];
  if (page >= 0 && page < a.pages) return page;
  report_error(a.err, ERR_BOUNDS, page);
  return -1;
}

// ---- one new token a sequence: D / 8 lanes for each (sequence, head) -----------------------------------------------------------------------------
// A decoding step moves a few hundred bytes a head, so what counts is the chain of dependent loads: the length beside the row, then the page, then its scale.
// 5.0 us for one sequence, 5.6 for 64 (48 query and 8 K/V heads of 128); the host takes 16 for the call.
template <typename T, bool F8>
__global__ void __launch_bounds__(128) paged_append_step_kernel(const __grid_constant__ PagedAppendArgs a) {
  pdl_entry();
  HeadLanes hl(a, threadIdx.x);
  const int heads = a.H + 2 * a.G, per = 128 / hl.lanes;
  const long long unit = static_cast<long long>(blockIdx.x) * per + threadIdx.x / hl.lanes;
  if (unit >= static_cast<long long>(a.B) * heads) return;
  const int b = static_cast<int>(unit / heads);
  int hd = static_cast<int>(unit % heads);
  if (a.q == nullptr && hd < a.H) return;
  const bool is_q = hd < a.H, is_v = hd >= a.H + a.G;
  if (!is_q) hd -= is_v ? a.H + a.G : a.H;
  const T* src = is_q ? static_cast<const T*>(a.q) + b * a.q_row + hd * a.q_head
                      : (is_v ? static_cast<const T*>(a.v) + b * a.v_row + hd * a.v_head : static_cast<const T*>(a.k) + b * a.k_row + hd * a.k_head);
  float f[8];
  pa_unpack8<T>(hl.raw(src), f);
  const NewRows nr = pa_new_rows(a, b);
  T* q_out = static_cast<T*>(a.q_out) + (static_cast<long long>(b) * a.H + hd) * a.D;
  if (nr.n == 0) {
    const float none[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (is_q) hl.store(q_out, none);
    return;
  }
  const int page = is_q ? 0 : pa_page(a, b, nr.first / a.P);
  if (page < 0) return;
  const long long at = static_cast<long long>(page) * a.G + hd;
  const int slot = nr.first % a.P;
  float* scales = is_v ? a.v_scale : a.k_scale;
  const float old = F8 && !is_q && slot > 0 ? scales[at] : 0.f;
  if (!is_v) {
    hl.turns(a, nr.first);
    hl.finish(a, static_cast<const T*>(is_q ? a.q_weight : a.k_weight), f);
  }
  if (is_q) {
    hl.store(q_out, f);
    return;
  }
  void* pages = is_v ? a.v_pages : a.k_pages;
  if constexpr (F8) {
    uint32_t m = pa_magnitude(f);
    for (int o = hl.lanes >> 1; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(hl.mask, m, o));
    const float want = pa_scale(m), scale = slot > 0 ? pa_joined(want, old) : want;
    uint8_t* tile = static_cast<uint8_t*>(pages) + at * a.P * a.D;
    if (slot > 0 && scale > old) {               // the older tokens in the new unit
      const float ratio = old / scale;
      for (int i = hl.lane * 16; i < slot * a.D; i += hl.lanes * 16) {
        uint4 u = *reinterpret_cast<uint4*>(tile + i);
        u.x = pa_recode4(u.x, ratio); u.y = pa_recode4(u.y, ratio); u.z = pa_recode4(u.z, ratio); u.w = pa_recode4(u.w, ratio);
        *reinterpret_cast<uint4*>(tile + i) = u;
      }
    }
    hl.store_codes(tile + slot * a.D, f, pa_inverse(scale));
    if (hl.lane == 0) scales[at] = scale;
  } else {
    hl.store(static_cast<T*>(pages) + (at * a.P + slot) * a.D, f);
  }
}

// ---- several new tokens a sequence ----------------------------------------------------------------------------------------------------------------
// The last of `n` steps whose bound is at most x: bounds rise from step to step, the first is at most x.  All threads of the block call it.
template <typename F>
__device__ __forceinline__ int pa_step_of(int n, long long x, F bound) {
  int at = 0;
  for (int base = 1; base < n; base += blockDim.x) {
    const int i = base + threadIdx.x;
    at += __syncthreads_count(i < n && bound(i) <= x);
  }
  return at;
}
// Units of a call's pages: sequence b has those from starts[b] / P + 2 b on; its rows touch at most (n - 2) / P + 2 pages.
__device__ __forceinline__ long long pa_first_unit(const PagedAppendArgs& a, int b) { return static_cast<long long>(a.starts[b]) / a.P + 2LL * b; }

constexpr int kQueryHeads = 8;             // of a row that D / 8 lanes take, four at a time: the rotation is read once for them

// One block per (page, head, keys or values) holds the page's new rows in registers between the maximum and the codes, IT vectors a thread; after the
// `page_units` of them, blocks for the queries.
template <typename T, bool F8, int IT>
__global__ void __launch_bounds__(IT == 8 ? 512 : 256, IT == 8 ? 1 : 4) paged_append_kernel(const __grid_constant__ PagedAppendArgs a, int page_units) {
  pdl_entry();
  HeadLanes hl(a, threadIdx.x);
  const int groups = blockDim.x / hl.lanes, group = threadIdx.x / hl.lanes;
  __shared__ uint32_t s_max[16];
  if (static_cast<int>(blockIdx.x) >= page_units) {
    const int chunks = (a.H + kQueryHeads - 1) / kQueryHeads;
    const long long item0 = (static_cast<long long>(blockIdx.x) - page_units) * groups, item = item0 + group;
    const int row = static_cast<int>(item / chunks), h0 = static_cast<int>(item % chunks) * kQueryHeads;
    int b = pa_step_of(a.B, item0 / chunks, [&](int i) { return static_cast<long long>(a.starts[i]); });
    if (row >= a.rows) return;
    while (b + 1 < a.B && a.starts[b + 1] <= row) ++b;
    const NewRows nr = pa_new_rows(a, b);
    const bool there = row >= nr.row && row < nr.row + nr.n;
    if (there) hl.turns(a, nr.first + row - nr.row);
    const T* src = static_cast<const T*>(a.q) + row * a.q_row;
    T* dst = static_cast<T*>(a.q_out) + static_cast<long long>(row) * a.H * a.D;
#pragma unroll
    for (int h = h0; h < h0 + kQueryHeads; h += 4) {
      uint4 raw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[i] = there && h + i < a.H ? hl.raw(src + (h + i) * a.q_head) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (h + i >= a.H) break;
        float f[8];
        pa_unpack8<T>(raw[i], f);
        if (there) hl.finish(a, static_cast<const T*>(a.q_weight), f);
        hl.store(dst + (h + i) * a.D, f);
      }
    }
    return;
  }
  const int unit = blockIdx.x / (2 * a.G), which = blockIdx.x % (2 * a.G), hd = which >> 1;
  const bool is_v = which & 1;
  const int b = pa_step_of(a.B, unit, [&](int i) { return pa_first_unit(a, i); });
  const NewRows nr = pa_new_rows(a, b);
  const long long j = nr.first / a.P + (unit - pa_first_unit(a, b));
  const int lo = static_cast<int>(max(static_cast<long long>(nr.first), j * a.P));
  const int hi = static_cast<int>(min(static_cast<long long>(nr.first) + nr.n, (j + 1) * a.P));
  if (nr.n == 0 || lo >= hi || j < 0) return;
  const int page = pa_page(a, b, static_cast<int>(j));
  if (page < 0) return;
  const long long at = static_cast<long long>(page) * a.G + hd;
  const int slot0 = lo - static_cast<int>(j) * a.P, row0 = nr.row + lo - nr.first, n = hi - lo;
  float f[IT][8];
  uint32_t m = 0;
  const T* src = is_v ? static_cast<const T*>(a.v) + row0 * a.v_row + hd * a.v_head : static_cast<const T*>(a.k) + row0 * a.k_row + hd * a.k_head;
  const long long step = is_v ? a.v_row : a.k_row;
  uint4 raw[IT];
#pragma unroll
  for (int it = 0; it < IT; ++it) raw[it] = it * groups + group < n ? hl.raw(src + (it * groups + group) * step) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int i = it * groups + group;
    pa_unpack8<T>(raw[it], f[it]);
    if (i < n) {
      if (!is_v) {
        hl.turns(a, lo + i);
        hl.finish(a, static_cast<const T*>(a.k_weight), f[it]);
      }
      m = max(m, pa_magnitude(f[it]));
    }
  }
  void* pages = is_v ? a.v_pages : a.k_pages;
  if constexpr (F8) {
    float* scales = is_v ? a.v_scale : a.k_scale;
    const float old = slot0 > 0 ? scales[at] : 0.f;
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) m = max(m, s_max[i]);
    const float want = pa_scale(m), scale = slot0 > 0 ? pa_joined(want, old) : want, inv = pa_inverse(scale);
    uint8_t* tile = static_cast<uint8_t*>(pages) + at * a.P * a.D;
    if (slot0 > 0 && scale > old) {
      const float ratio = old / scale;
      for (int i = threadIdx.x * 16; i < slot0 * a.D; i += blockDim.x * 16) {
        uint4 u = *reinterpret_cast<uint4*>(tile + i);
        u.x = pa_recode4(u.x, ratio); u.y = pa_recode4(u.y, ratio); u.z = pa_recode4(u.z, ratio); u.w = pa_recode4(u.w, ratio);
        *reinterpret_cast<uint4*>(tile + i) = u;
      }
    }
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int i = it * groups + group;
      if (i < n) hl.store_codes(tile + (slot0 + i) * a.D, f[it], inv);
    }
    if (threadIdx.x == 0) scales[at] = scale;
  } else {
    T* tile = static_cast<T*>(pages) + at * a.P * a.D;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int i = it * groups + group;
      if (i < n) hl.store(tile + (slot0 + i) * a.D, f[it]);
    }
  }
}

template <typename T, bool F8>
int paged_append_launch(const PagedAppendArgs& a, cudaStream_t stream) {
  const int lanes = a.D / 8;
  if (a.starts == nullptr) {
    const long long units = static_cast<long long>(a.B) * (a.H + 2 * a.G);
    return (int)launch_dependent(paged_append_step_kernel<T, F8>, dim3(static_cast<unsigned>((units * lanes + 127) / 128)), dim3(128), 0, stream, a);
  }
  // every sequence takes rows / P + 2 units at most
  const int vectors = a.P * lanes, threads = vectors > 2048 ? 512 : vectors > 128 ? 256 : 128;
  const long long units = (static_cast<long long>(a.rows) / a.P + 2LL * a.B) * 2 * a.G;
  const long long queries = a.q ? static_cast<long long>(a.rows) * ((a.H + kQueryHeads - 1) / kQueryHeads) : 0, blocks = units + (queries + threads / lanes - 1) / (threads / lanes);
  if (blocks > 0x7fffffffLL) return -5;
  const dim3 grid(static_cast<unsigned>(blocks)), block(threads);
  const int u = static_cast<int>(units);
  switch ((vectors + threads - 1) / threads) {
    case 1: return (int)launch_dependent(paged_append_kernel<T, F8, 1>, grid, block, 0, stream, a, u);
    case 2: return (int)launch_dependent(paged_append_kernel<T, F8, 2>, grid, block, 0, stream, a, u);
    case 4: return (int)launch_dependent(paged_append_kernel<T, F8, 4>, grid, block, 0, stream, a, u);
    case 8: return (int)launch_dependent(paged_append_kernel<T, F8, 8>, grid, block, 0, stream, a, u);
  }
  return -6;
}

}  // namespace tyr

using namespace tyr;

// dtype: 0 = bf16, 1 = fp16 (operands, and pages without scales)
extern "C" TYR_EXPORT int tyr_paged_append(const void* packed, int dtype, void* stream) {
  const PagedAppendArgs& a = *static_cast<const PagedAppendArgs*>(packed);
  if (a.rows <= 0 || a.B <= 0 || a.H < 0 || a.G <= 0 || a.pages <= 0 || a.width <= 0) return -1;
  if ((a.D != 64 && a.D != 128 && a.D != 256) || (a.P != 16 && a.P != 32 && a.P != 64 && a.P != 128)) return -2;
  if (a.half < 0 || a.half % 4 != 0 || 2 * a.half > a.D || (a.half > 0 && (a.cos == nullptr || a.sin == nullptr))) return -3;
  if ((a.q != nullptr) != (a.q_out != nullptr) || (a.k_scale != nullptr) != (a.v_scale != nullptr)) return -4;
  const bool f8 = a.k_scale != nullptr;
  if (dtype == 0) return f8 ? paged_append_launch<__nv_bfloat16, true>(a, (cudaStream_t)stream) : paged_append_launch<__nv_bfloat16, false>(a, (cudaStream_t)stream);
  if (dtype == 1) return f8 ? paged_append_launch<__half, true>(a, (cudaStream_t)stream) : paged_append_launch<__half, false>(a, (cudaStream_t)stream);
  return -7;
}
