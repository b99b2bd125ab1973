// Attention of new tokens over a paged cache, in 16 bits or as e4m3 codes with a scale for each (page, head) (csrc/paged_append.cu writes it).
//
// Sequence b has lengths[b] tokens in pages table[b, ..], the last n of which are the call's rows (n = 1 without starts); row i sees the positions up to its
// own, the last `window` of them where one is given.  The R = H / G query heads of a K/V head share its keys: a row of the products is a (token, head) pair.
//
//   s = scale q.k,   m = max s,   l = sum 2^(s - m),   out = sum 2^(s - m) v / l          (s in units of log2 e)
//
// Bound: the keys and values are read once, 2 D bytes a (key, head) in e4m3, for 4 R D operations; up to some hundred operations a byte the memory bounds it.
//
// One producer warp copies tiles of keys and values by TMA into a ring of stages (page by page, 128-byte swizzle), four consumer warps multiply with
// mma.sync m16n8k16: either every warp takes tiles of its own (32 keys of 128 bytes) for the same 16 rows (ROWS 16: decoding, the warps' results are joined through shared
// memory), or 16 of 128 rows (of 64 with heads of 256) for all tiles of 64 keys (several new tokens).
//
// Every operand comes from shared memory in 16-byte pieces: the order of the channels within a product's sum is free as long as the queries follow it, and so is
// the order of the keys as long as the values follow it.  The keys and the values are the products' first operands (16 of them, or 16 channels, by 8 rows; a second
// 8 rows where there are more), so that few rows leave nothing idle but columns.  A lane (g, t) reads bytes 16 t .. 16 t + 15 (and every 64 on) of key row pi(g), pi(n) = n for even n
// and n ^ 4 for odd n, and channels 16 g .. 16 g + 15 of the four value rows that its probabilities belong to; with the swizzle neither conflicts.
//
// e4m3 becomes f16 two codes at a time (64 lanes a clock an SM, as the byte permutes that pair the values' rows; done by masks and shifts it took three operations
// and bound the kernel).  Queries in bf16 are scaled by a power of two for each row into f16's range.  With M = max (s + log2 v_scale) beside m, the probabilities
// times the page's value scale stay below f16's upper end whatever the scales: 2^(s + log2 v_scale - M), and the result is taken times 2^(M - m) / l.  At the lower end
// they keep all their bits down to 2^-22 of a row's largest such product and are nothing below 2^-33: beside a page with a scale some million times another's, that
// one's values lose bits in every channel.
//
// Work is cut into equal shares of tiles, one for each resident CTA, whatever the lengths: a share may begin and end inside a (sequence, head).  Such pieces go to
// a workspace of the call, and a second launch joins them in the order of the keys.
//
// Measured, e4m3: 32 sequences of some 16 000 tokens, 48 query heads over 8 of 128: 137 us and 7 for the join, 5.7 TB/s, while it streams 93 % of what a copy moves.
// 32 of some 2000, 24 heads over 4 of 256: 31.6 us, of which 4 pass before the first keys arrive (the shares are found from the lengths) and 5 in the join; two CTAs
// of five warps are what 168 registers leave room for.  One of 500: 8.6 us and 4.6.  The join is a launch of its own: the last CTA to
// end would need a counter that each call clears, and two replayed graphs would share it.
#include <type_traits>

#include "common.cuh"
#include "per_device.h"

namespace tyr {

// keys of a tile: while decoding some 8 KB of keys and values, a warp's own
__host__ __device__ constexpr int tile_keys(int rows, int row_bytes) { return rows > 16 ? 64 : row_bytes <= 128 ? 32 : 16; }
// Consumer warps of a form: 16 rows each, or four with the same 16.
__host__ __device__ constexpr int warps_of(int rows) { return rows == 16 ? 4 : rows / 16; }

struct PagedAttnArgs {
  const void* q;                               // [rows, H, D]; element strides below
  void* out;                                   // [rows, H, D]
  const void *k_pages, *v_pages;               // [pages, G, P, D]
  const float *k_scale, *v_scale;              // [pages, G] (null: 16-bit pages)
  const int *table, *lengths, *starts;         // [B, width], [B], [B + 1] (nullable)
  float* part;                                 // workspace (see part_stats)
  int* err;
  long long q_row, q_head, table_row;
  int rows, B, H, G, D, P, pages, width, window, whole;       // P: 16, 32, 64 or 128
  float scale;
  int ctas;                                    // shares of the work that `part` has room for (not read where shares are whole items)
};
static_assert(sizeof(PagedAttnArgs) == 160, "as ops/paged_cache.py packs it");

struct PartHead { int row, heads, used, last, slot, pad[3]; };      // a (sequence, head, row tile) that begins in this CTA's share and ends in CTA `last`'s

struct Seq { int row, n, len, tile0, tiles, row_tiles; };

// Rows row .. end - 1 that sequence b brings, and whether they go together with its length, the table and the call.
struct Rows { int row, end, len; bool fits; };
__device__ __forceinline__ Rows rows_of(const PagedAttnArgs& a, int b) {
  Rows r;
  r.len = a.lengths[b];
  r.row = a.starts ? a.starts[b] : b;
  r.end = a.starts ? a.starts[b + 1] : b + (r.len > 0 ? 1 : 0);
  r.fits = r.row == r.end || (r.row >= 0 && r.row < r.end && r.end <= a.rows && r.len >= r.end - r.row && (r.len - 1) >> (31 - __clz(a.P)) < a.width);
  return r;
}
// Rows, keys and tiles of sequence b; none where the operands do not go together (recorded).
template <int ROWS, int KEYS>
__device__ __forceinline__ Seq seq_of(const PagedAttnArgs& a, int b) {
  Seq s;
  const Rows r = rows_of(a, b);
  s.len = r.len;
  s.row = r.row;
  s.n = r.fits ? r.end - r.row : 0;
  if (!r.fits) report_error(a.err, ERR_BOUNDS, b);
  const int first = a.window > 0 ? max(0, s.len - s.n - a.window + 1) : 0;
  s.tile0 = first / KEYS;
  s.tiles = s.n == 0 ? 0 : (s.len + KEYS - 1) / KEYS - s.tile0;
  s.row_tiles = s.n == 0 ? 0 : (s.n * (a.H / a.G) + ROWS - 1) / ROWS;
  return s;
}
__device__ __forceinline__ int seq_work(const PagedAttnArgs& a, const Seq& s) { return a.G * s.row_tiles * (a.whole ? 1 : s.tiles); }

__device__ __forceinline__ long long warp_sum64(long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// This CTA's share of the work, walked piece by piece: a piece is a run of tiles of one (sequence, head, row tile).  Every warp walks it for itself.
template <int ROWS, int KEYS>
struct Share {
  const PagedAttnArgs& a;
  long long at, end, before, per;              // in tiles (items where shares are whole items); `before`: work of the sequences before b
  int b, lane;
  Seq s;
  int head, row_tile, x0, x1, first, last;     // the piece: tiles first .. last - 1 that its rows see, x0 .. x1 of the item's
  bool begins, ends;
  long long item_end;

  __device__ __forceinline__ Share(const PagedAttnArgs& args, int lane_) : a(args), lane(lane_) {
    const long long first_work = lane < a.B ? seq_work(a, seq_of<ROWS, KEYS>(a, lane)) : 0;
    long long sum = first_work;
    for (int i = lane + 32; i < a.B; i += 32) sum += seq_work(a, seq_of<ROWS, KEYS>(a, i));
    const long long total = warp_sum64(sum);
    per = total >> 31 ? (total + gridDim.x - 1) / gridDim.x : (static_cast<uint32_t>(total) + gridDim.x - 1) / gridDim.x;
    at = min(static_cast<long long>(blockIdx.x) * per, total);
    end = min(at + per, total);
    before = 0;
    b = 0;
    if (at >= end) return;
    for (int base = 0; base < a.B; base += 32) {
      const long long mine = base == 0 ? first_work : base + lane < a.B ? seq_work(a, seq_of<ROWS, KEYS>(a, base + lane)) : 0;
      long long upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, before + upto > at);
      if (past) {
        const int l = __ffs(past) - 1;
        b = base + l;
        before += __shfl_sync(0xffffffffu, upto - mine, l);
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    s = seq_of<ROWS, KEYS>(a, b);
  }
  __device__ __forceinline__ bool next() {
    if (at >= end) return false;
    while (at - before >= seq_work(a, s)) {
      before += seq_work(a, s);
      if (++b >= a.B) return false;
      s = seq_of<ROWS, KEYS>(a, b);
    }
    const int off = static_cast<int>(at - before), unit = a.whole ? 1 : s.tiles, item = off / unit;
    head = item / s.row_tiles;
    row_tile = item - head * s.row_tiles;
    x0 = off - item * unit;
    const long long left = end - at;
    x1 = left < unit - x0 ? x0 + static_cast<int>(left) : unit;
    item_end = at - x0 + unit;
    begins = x0 == 0;
    ends = x1 == unit;
    at += x1 - x0;
    // tiles that the piece's rows see
    const int R = a.H / a.G, held = s.len - s.n, i0 = row_tile * ROWS / R, i1 = min(s.n, (row_tile * ROWS + ROWS - 1) / R + 1) - 1;
    const int lo = a.window > 0 ? max(0, held + i0 - a.window + 1) : 0;
    first = lo / KEYS;
    last = (held + i1) / KEYS + 1;
    if (!a.whole) {
      first = max(first, s.tile0 + x0);
      last = min(last, s.tile0 + x1);
    }
    return true;
  }
};

template <bool F8, int D, int KEYS>
struct Tile {
  static constexpr int kBytes = F8 ? 1 : 2;
  static constexpr int kRow = D * kBytes < 128 ? D * kBytes : 128;          // bytes of a row in a box
  static constexpr int kBoxes = D * kBytes / kRow;
  static constexpr int kSize = KEYS * D * kBytes;                          // of the keys, and of the values
  static constexpr int kChunks = D * kBytes / 16;
  static constexpr int kRun = F8 && D >= 128 ? 16 : 8;                      // channels of a box that a lane takes of a value row
  // 16-byte piece c of row r
  static __device__ __forceinline__ uint32_t at(uint32_t base, int r, int c) {
    constexpr int per = kRow / 16;
    const int swizzle = kRow == 128 ? r & 7 : (r >> 1) & 3;
    return base + (c / per) * (KEYS * kRow) + r * kRow + (((c % per) ^ swizzle) << 4);
  }
};

// Registers and shared memory of a form.  A CTA has five warps, and each quarter of an SM 16384 registers: three CTAs fit with 128 a thread, two (or one of nine
// warps) with 168, one with more; the fewer stages that many CTAs leave are enough while there are two.
template <bool F8, int D, int ROWS, int NR>
struct Form {
  static constexpr int kKeys = tile_keys(ROWS, D * (F8 ? 1 : 2));
  using TL = Tile<F8, D, kKeys>;
  static constexpr int kWarps = warps_of(ROWS), kThreads = (kWarps + 1) * 32;
  static constexpr bool kQueriesInRegisters = D == 64 || (D == 128 && ROWS == 16);
  static constexpr int kExtra = 1024 + 1024 + (kQueriesInRegisters ? 0 : (ROWS == 16 ? 1 : kWarps) * (D / 16) * 512) + (ROWS == 16 ? kWarps * 8 * NR * 32 * 4 : 0);
  // ROWS 16: a multiple of the warps, so that a stage is always the same warp's.  A warp that waits for a stage's next use has then seen its last one, and one bit
  // tells them apart.
  static constexpr int stages(int ctas) {
    const int n = ((227 * 1024) / ctas - 1024 - kExtra) / (2 * TL::kSize + 48);
    return ROWS == 16 ? n / kWarps * kWarps : n;
  }
  static constexpr int kFew = ROWS == 16 ? 2 * kWarps : 2;                  // one in use and one on its way
  static constexpr int kWanted = ROWS > 16 ? 1 : D == 64 ? 3 : (NR == 1 ? (D == 128 ? 3 : 2) : (D == 128 ? 2 : 1));
  static constexpr int kCtas = stages(kWanted) >= kFew ? kWanted : (kWanted > 1 && stages(kWanted - 1) >= kFew ? kWanted - 1 : 1);
  static constexpr int kStages = stages(kCtas) < 12 ? stages(kCtas) : 12;
  static_assert(kStages >= kFew, "shared memory");
  static constexpr int kSmem = kExtra + kStages * (2 * TL::kSize + 48);
  static constexpr int kBound = kWarps == 8 ? 384 : kCtas == 3 ? 256 : (kCtas == 2 ? 192 : 160);      // threads of which two CTAs (or one) share the registers
  static constexpr int kAtOnce = kCtas == 1 ? 1 : 2;
};

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t pt_prmt(uint32_t x, uint32_t y, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(y), "r"(sel));
  return r;
}
// the two codes in a word's lower half -> two halves
__device__ __forceinline__ uint32_t halves_of_codes(uint32_t w) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(w)));
  return r;
}

template <typename T> struct Num;
template <> struct Num<__nv_bfloat16> {
  static constexpr uint32_t kExponent = 0x7f80u;
  static __device__ __forceinline__ float2 two(uint32_t u) { return unpack_bf16x2(u); }
  static __device__ __forceinline__ uint32_t pack(float x, float y) { return pack_bf16x2(x, y); }
};
template <> struct Num<__half> {
  static constexpr uint32_t kExponent = 0x7c00u;
  static __device__ __forceinline__ float2 two(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
// Infinities and NaN among a word's two numbers of type T: an exponent of ones carries into the sign's place.
template <typename T> __device__ __forceinline__ uint32_t odd_bits(uint32_t w) {
  constexpr uint32_t kOnes = Num<T>::kExponent * 0x10001u, kLast = __is_same(T, __half) ? 0x04000400u : 0x00800080u;
  return (w & kOnes) + kLast;
}
template <typename T> __device__ __forceinline__ bool any_odd(const uint4& u) {
  return ((odd_bits<T>(u.x) | odd_bits<T>(u.y) | odd_bits<T>(u.z) | odd_bits<T>(u.w)) & 0x80008000u) != 0u;
}
// Zeros in their place; whether there were any.
template <typename T>
__device__ __forceinline__ bool without_odd(uint4& u) {
  bool any = false;
  uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t odd = odd_bits<T>(w[i]);
    if (odd & 0x8000u) w[i] &= 0xffff0000u;
    if (odd & 0x80000000u) w[i] &= 0xffffu;
    any |= (odd & 0x80008000u) != 0u;
  }
  u = make_uint4(w[0], w[1], w[2], w[3]);
  return any;
}
// c [16, 8] += a [16, 16] b [16, 8]; M is the operands' type.
template <typename M>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (__is_same(M, __half)) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}
// An 8 x 8 matrix of 16-bit numbers, a lane (g, t) holding row g's 2 t and 2 t + 1, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

__device__ __forceinline__ float pt_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The workspace holds, for each of `ctas` shares, the head of its split item (8 floats) and two pieces of ROWS rows: {m, l, M, -} and D sums each.
__device__ __forceinline__ float* part_stats(const PagedAttnArgs& a, int ctas, int rows, int piece) { return a.part + ctas * 8LL + static_cast<long long>(piece) * rows * 4; }
__device__ __forceinline__ float* part_sums(const PagedAttnArgs& a, int ctas, int rows, int piece) {
  return a.part + ctas * 8LL + 2LL * ctas * rows * 4 + static_cast<long long>(piece) * rows * a.D;
}

template <typename T>
__device__ __forceinline__ void write4(T* p, float4 v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(Num<T>::pack(v.x, v.y), Num<T>::pack(v.z, v.w));
}

// Values that are not finite at keys that not all rows of a piece see, to the result (or the piece's sums) of those that do: once more through this CTA's share, when all of
// it is written.  A call of its own, so that the products' registers are none of its: among the products it took up to a quarter of every call.
template <typename T, int D, int ROWS, int KEYS>
__device__ __noinline__ void add_odd(const PagedAttnArgs& a) {
  Share<ROWS, KEYS> sh(a, threadIdx.x & 31);
  const int R = a.H / a.G;
  for (int slot = 0; sh.next(); slot = 1) {
    const int held = sh.s.len - sh.s.n, used = min(ROWS, sh.s.n * R - sh.row_tile * ROWS), p0 = held + sh.row_tile * ROWS / R, p1 = held + (sh.row_tile * ROWS + used - 1) / R;
    const int seen0 = a.window > 0 ? max(0, p1 - a.window + 1) : 0, seen1 = p0 + 1;      // keys that all rows see went through the products; adding others twice is the same
    for (int i = threadIdx.x; i < used * D; i += blockDim.x) {
      const int in_tile = i / D, d = i % D, row = sh.row_tile * ROWS + in_tile, p = held + row / R;
      for (int key = max(sh.first * KEYS, a.window > 0 ? p - a.window + 1 : 0); key < min(sh.last * KEYS, p + 1); ++key) {
        if (key >= seen0 && key < seen1) {
          key = seen1 - 1;
          continue;
        }
        const int page = a.table[sh.b * a.table_row + key / a.P];
        if (page < 0 || page >= a.pages) continue;
        const T v = static_cast<const T*>(a.v_pages)[((static_cast<long long>(page) * a.G + sh.head) * a.P + key % a.P) * D + d];
        if ((odd_bits<T>(reinterpret_cast<const uint16_t&>(v)) & 0x8000u) == 0u) continue;
        if (sh.begins && sh.ends) {
          T& out = static_cast<T*>(a.out)[((sh.s.row + static_cast<long long>(row / R)) * a.H + sh.head * R + row % R) * D + d];
          out = static_cast<T>(static_cast<float>(out) + static_cast<float>(v));
        } else {
          part_sums(a, gridDim.x, ROWS, 2 * blockIdx.x + slot)[static_cast<long long>(in_tile) * D + d] += static_cast<float>(v);
        }
      }
    }
  }
}

// T: type of the queries, the results and 16-bit pages; NR: rows of a lane (1: at most 8 rows in a tile of 16).
template <typename T, bool F8, int D, int ROWS, int NR>
__global__ void __launch_bounds__(Form<F8, D, ROWS, NR>::kBound, Form<F8, D, ROWS, NR>::kAtOnce) paged_attention_kernel(const __grid_constant__ PagedAttnArgs a, const __grid_constant__ CUtensorMap map_k,
                                                                           const __grid_constant__ CUtensorMap map_v) {
  constexpr int KEYS = Form<F8, D, ROWS, NR>::kKeys;
  using TL = Tile<F8, D, KEYS>;
  using M = typename std::conditional<F8, __half, T>::type;                 // operands of the products
  using FM = Form<F8, D, ROWS, NR>;
  constexpr int kWarps = FM::kWarps, kSync = kWarps * 32;                   // threads that meet at the consumers' barrier
  constexpr int STAGES = FM::kStages, KSTEPS = D / 16, TILES = D / 16;
  constexpr int GROUPS = KEYS / 16;                                         // runs of 16 keys
  constexpr bool QREG = FM::kQueriesInRegisters;                                           // the queries' fragments stay in registers
  constexpr float kShift = 8.f;                                             // probabilities times 2^8: further from f16's small end
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* extra = smem + STAGES * 2 * TL::kSize;
  float2* s_scale = reinterpret_cast<float2*>(extra);                       // [STAGES][4]: scale of the keys, log2 of the values'
  volatile int* met_odd = reinterpret_cast<volatile int*>(extra);             // 16-bit pages, which have no scales: whether values that are not finite were met
  uint64_t* full = reinterpret_cast<uint64_t*>(extra + STAGES * 32);
  uint64_t* empty = full + STAGES;
  float* s_stats = reinterpret_cast<float*>(empty + STAGES);                // [4][16][4], joining warps (ROWS 16)
  uint4* s_q = reinterpret_cast<uint4*>(s_stats + 256);                     // fragments of the queries, QREG false: [warps that differ][KSTEPS][32]
  float* s_sum = reinterpret_cast<float*>(s_q + (QREG ? 0 : (ROWS == 16 ? 1 : kWarps) * KSTEPS * 32));   // [4][8 NR][32] (ROWS 16)

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, ROWS == 16 ? 1 : kWarps);
    }
    mbar_fence_init();
    if (!F8) *met_odd = 0;
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  __syncthreads();
  pdl_wait();
  const int R = a.H / a.G;
  Share<ROWS, KEYS> sh(a, lane);
  uint32_t turn = 0;                                                        // tiles before this one: its stage and the parity of the stage's use

  if (warp == kWarps) {
    // ---- producer ---------------------------------------------------------------------------------------------------
    const int page_rows = min(a.P, KEYS), page_bits = 31 - __clz(a.P), per_tile = KEYS >> min(page_bits, 31 - __clz(KEYS));
    for (bool ok = true; ok && sh.next();) {
      const int last_page = (sh.s.len - 1) >> page_bits;
      const int* table = a.table + sh.b * a.table_row;
      int batch = -1, id = 0;                       // pages 32 batch .. of the sequence, one a lane
      float2 scale = make_float2(1.f, 0.f);
      for (int tile = sh.first; tile < sh.last; ++tile, ++turn) {
        const int stage = turn % STAGES, phase = turn / STAGES & 1;
        const int p0 = tile * KEYS >> page_bits;
        if (p0 >> 5 != batch) {
          batch = p0 >> 5;
          const int p = batch * 32 + lane;
          id = p <= last_page ? table[p] : 0;
          scale = make_float2(1.f, 0.f);
          if (id < 0 || id >= a.pages) {                                    // outside the cache: nothing is read, and the keys are no numbers
            report_error(a.err, ERR_BOUNDS, id);
            id = -1;
            scale.x = __uint_as_float(0x7fffffffu);
          } else if (F8) {
            scale = make_float2(a.k_scale[static_cast<long long>(id) * a.G + sh.head], log2f(a.v_scale[static_cast<long long>(id) * a.G + sh.head]));
          }
        }
        const int n = min(per_tile, last_page - p0 + 1), from = (p0 & 31) + lane;
        const int page = __shfl_sync(0xffffffffu, id, from & 31);
        const float2 sc = make_float2(__shfl_sync(0xffffffffu, scale.x, from & 31), __shfl_sync(0xffffffffu, scale.y, from & 31));
        if (!mbar_wait(empty + stage, phase ^ 1, a.err, 1)) {
          ok = false;
          break;
        }
        if (F8 && lane < per_tile) s_scale[stage * 4 + lane] = sc;
        __syncwarp();
        if (lane == 0) mbar_expect_tx(full + stage, static_cast<uint32_t>(2 * n * page_rows * D * TL::kBytes));
        __syncwarp();
        if (lane < n) {
          uint8_t* dst = smem + stage * 2 * TL::kSize + lane * page_rows * TL::kRow;
          const int row = (tile * KEYS) & (a.P - 1), z = page < 0 ? -1 : page * a.G + sh.head;      // -1: what the map fills in
          if (TL::kBoxes == 1 || per_tile == 1) {                           // all columns at once: they lie as the tile has them
            tma_load_4d(dst, &map_k, full + stage, 0, row, 0, z);
            tma_load_4d(dst + TL::kSize, &map_v, full + stage, 0, row, 0, z);
          } else {
#pragma unroll
            for (int c = 0; c < TL::kBoxes; ++c) {
              tma_load_4d(dst + c * KEYS * TL::kRow, &map_k, full + stage, 0, row, c, z);
              tma_load_4d(dst + TL::kSize + c * KEYS * TL::kRow, &map_v, full + stage, 0, row, c, z);
            }
          }
        }
      }
    }
    // rows of no sequence, and of those whose operands do not go together
    const auto clear = [&](int row) {
      for (int i = lane * 8; i < a.H * D; i += 256) *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + static_cast<long long>(row) * a.H * D + i) = make_uint4(0u, 0u, 0u, 0u);
    };
    for (int row = blockIdx.x; row < a.rows; row += gridDim.x)
      if (a.starts ? row < a.starts[0] || row >= a.starts[a.B] : a.lengths[row] <= 0 || !rows_of(a, row).fits) clear(row);
    if (a.starts)
      for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
        const Rows r = rows_of(a, b);
        if (!r.fits)
          for (int row = max(r.row, 0); row < min(r.end, a.rows); ++row) clear(row);
      }
    if constexpr (!F8) {
      __syncthreads();
      if (*met_odd != 0) add_odd<T, D, ROWS, KEYS>(a);
    }
    return;
  }

  // ---- consumers ------------------------------------------------------------------------------------------------------
  const int page_bits = 31 - __clz(a.P);
  const int g = lane >> 2, t = lane & 3, pi = g & 1 ? g ^ 4 : g;
  const int tid = threadIdx.x;
  // this lane's pieces of a tile: rows 8 apart and boxes lie the same way
  constexpr int PIECES_BOX = TL::kRow / 64;                                 // of a key row in a box
  uint32_t k_at[PIECES_BOX], v_at[2];
#pragma unroll
  for (int c = 0; c < PIECES_BOX; ++c) k_at[c] = TL::at(0, pi, t + 4 * c);
#pragma unroll
  for (int i = 0; i < 2; ++i) v_at[i] = F8 && D == 64 ? TL::at(0, i ? (2 * t + 1) ^ 4 : 2 * t, g >> 1) + (g & 1) * 8 : TL::at(0, i ? (2 * t + 1) ^ 4 : 2 * t, g);
  PartHead head{0, 0, 0, -1, 0, {0, 0, 0}};
  if (tid == 0 && !a.whole) *reinterpret_cast<PartHead*>(a.part + blockIdx.x * 8LL) = head;
  bool first_piece = true, lost = false;
  while (sh.next()) {
    const int held = sh.s.len - sh.s.n, used = min(ROWS, sh.s.n * R - sh.row_tile * ROWS);         // rows of this tile
    const int warp_row = ROWS == 16 ? 0 : warp * 16;
    // ---- queries: row g (and g + 8) in fragments; the scores' rows are 2 t and 2 t + 1 (and 8 further) ----------------------------
    uint32_t qa[QREG ? KSTEPS : 1][2 * NR];
    float factor[NR];
    if (!QREG) asm volatile("bar.sync 1, %0;" ::"n"(kSync) : "memory");                // the last piece's fragments are no longer read
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int in_tile = warp_row + g + 8 * r, row = sh.row_tile * ROWS + in_tile, i = row / R;
      const bool there = in_tile < used;
      const T* src = static_cast<const T*>(a.q) + (there ? (sh.s.row + i) * a.q_row + (sh.head * R + row % R) * a.q_head : 0);
      constexpr int PIECES = TL::kChunks / 4;                                // 16-byte pieces of a key row that a lane takes
      constexpr int PER = F8 ? 16 : 8;                                       // channels of one
      uint32_t raw[PIECES][PER / 2];
#pragma unroll
      for (int c = 0; c < PIECES; ++c)
#pragma unroll
        for (int e = 0; e < PER / 8; ++e) {
          const uint4 u = there ? *reinterpret_cast<const uint4*>(src + PER * (t + 4 * c) + 8 * e) : make_uint4(0u, 0u, 0u, 0u);
          raw[c][4 * e] = u.x; raw[c][4 * e + 1] = u.y; raw[c][4 * e + 2] = u.z; raw[c][4 * e + 3] = u.w;
        }
      factor[r] = a.scale * 1.4426950408889634f;
      if constexpr (F8) {
        float up = 1.f;
        if constexpr (!__is_same(T, __half)) {                               // bf16 to f16: the row's largest magnitude to 1 .. 2
          float top = 0.f;
#pragma unroll
          for (int c = 0; c < PIECES; ++c)
#pragma unroll
            for (int e = 0; e < PER / 2; ++e) {
              const float2 v = Num<T>::two(raw[c][e]);
              top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
            }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -100), 100);
          up = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
          factor[r] *= __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        }
        const uint32_t* flat = &raw[0][0];
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks) {
          uint32_t x = flat[2 * ks], y = flat[2 * ks + 1];
          if constexpr (!__is_same(T, __half)) {
            const float2 u = Num<T>::two(x), v = Num<T>::two(y);
            x = Num<__half>::pack(u.x * up, u.y * up);
            y = Num<__half>::pack(v.x * up, v.y * up);
          }
          if constexpr (QREG) {
            qa[ks][r] = x;
            qa[ks][NR + r] = y;
          } else if (ROWS != 16 || warp == 0) {
            uint32_t* dst = reinterpret_cast<uint32_t*>(s_q + ((ROWS == 16 ? 0 : warp) * KSTEPS + ks) * 32 + lane);
            dst[r] = x;
            dst[NR + r] = y;
          }
        }
      } else {
        const uint32_t* flat = &raw[0][0];
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks) {
          if constexpr (QREG) {
            qa[ks][r] = flat[2 * ks];
            qa[ks][NR + r] = flat[2 * ks + 1];
          } else if (ROWS != 16 || warp == 0) {
            uint32_t* dst = reinterpret_cast<uint32_t*>(s_q + ((ROWS == 16 ? 0 : warp) * KSTEPS + ks) * 32 + lane);
            dst[r] = flat[2 * ks];
            dst[NR + r] = flat[2 * ks + 1];
          }
        }
      }
    }
    if (!QREG) asm volatile("bar.sync 1, %0;" ::"n"(kSync) : "memory");
    float by_row[NR][2];                                                     // of the scores' rows
    int pos[NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int in_tile = warp_row + 8 * r + 2 * t + e;
        by_row[r][e] = __shfl_sync(0xffffffffu, factor[r], (2 * t + e) * 4);
        pos[r][e] = in_tile < used ? held + (sh.row_tile * ROWS + in_tile) / R : -1;
      }
    // every key of tiles from `clear0` to before `clear1` is seen by all rows of the piece
    const int p_first = held + sh.row_tile * ROWS / R, p_last = held + (sh.row_tile * ROWS + used - 1) / R;
    const int clear0 = a.window > 0 ? (max(0, p_last - a.window + 1) + KEYS - 1) / KEYS : 0, clear1 = (p_first + 1) / KEYS;

    const int p_warp = held + (sh.row_tile * ROWS + min(used, warp_row + 16) - 1) / R;
    // keys that all of this warp's rows see: from seen0 on, before seen1
    const int seen0 = a.window > 0 ? max(0, p_warp - a.window + 1) : 0, seen1 = held + (sh.row_tile * ROWS + warp_row) / R + 1;

    float m[NR][2], l[NR][2], top[NR][2], o[TILES][NR][4];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) m[r][e] = top[r][e] = -INFINITY, l[r][e] = 0.f;
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][r][e] = 0.f;

    // ROWS 16: every fourth tile of all
    const uint32_t first_turn = turn;
    const int skip = ROWS == 16 ? static_cast<int>((warp - first_turn) & (kWarps - 1)) : 0, step = ROWS == 16 ? kWarps : 1;
    for (int tile = sh.first + skip; tile < sh.last; tile += step) {
      turn = first_turn + (tile - sh.first);
      const int stage = turn % STAGES;
      if (lost || !mbar_wait(full + stage, turn / STAGES & 1, a.err, 2)) {
        lost = true;                                                        // recorded; the warps still meet at their barriers
        break;
      }
      if (ROWS > 16 && (warp_row >= used || tile * KEYS > p_warp)) {        // nothing that this warp's rows see
        if (lane == 0) mbar_arrive(empty + stage);
        continue;
      }
      const uint32_t kb = smem_u32(smem + stage * 2 * TL::kSize), vb = kb + TL::kSize;
      const int key0 = tile * KEYS;
      const bool masked = tile < clear0 || tile >= clear1;
      // Values that are not finite at keys that not all of the warp's rows see: an unseen one times a probability of 0 would be NaN.  They become zeros in place, by every warp for itself
      // (all write the same), and are added to the result of the rows that see them.  Looking takes 88 -> 92 us of 6 x 64 tokens of 20 heads over 3000 tokens of 4, and
      // nothing while decoding, where every row sees all keys.
      if constexpr (!F8) {
        if (masked) {
          const int n = min(KEYS, sh.s.len - key0), past = min(n, max(0, seen1 - key0)), ahead = min(past, seen0 - key0);      // keys before `ahead`, and from `past` on
          const auto unseen = [&](auto f) {
#pragma unroll 1
            for (int i = lane; i < ahead * TL::kChunks; i += 32) f(TL::at(vb, i / TL::kChunks, i % TL::kChunks));
#pragma unroll 1
            for (int i = past * TL::kChunks + lane; i < n * TL::kChunks; i += 32) f(TL::at(vb, i / TL::kChunks, i % TL::kChunks));
          };
          bool odd = false;
          unseen([&](uint32_t at) { odd |= any_odd<T>(lds128(at)); });
          if (__any_sync(0xffffffffu, odd)) {
            *met_odd = 1;
            __threadfence_block();                                          // whoever finds zeros finds this
            unseen([&](uint32_t at) {
              uint4 u = lds128(at);
              if (without_odd<T>(u)) sts128(at, u);
            });
            fence_proxy_async();                                            // before the stage's next copy
            __syncwarp();
          }
        }
      }
      // ---- scores: keys pi(g) and pi(g) + 8 of every 16, rows 2 t and 2 t + 1 --------------------------------------------------
      // one run of keys and rows: its products in two sums, each half as long a chain
      constexpr int CHAINS = GROUPS * NR == 1 ? 2 : 1;
      float s[GROUPS][NR][4], s_odd[CHAINS][4];
#pragma unroll
      for (int j = 0; j < GROUPS; ++j)
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[j][r][e] = s_odd[0][e] = 0.f;
#pragma unroll
      for (int c = 0; c < TL::kChunks / 4; ++c) {
        constexpr int STEPS = F8 ? 4 : 2;
        uint32_t qs[STEPS][2 * NR];
#pragma unroll
        for (int w = 0; w < STEPS; ++w) {
          if constexpr (QREG) {
#pragma unroll
            for (int e = 0; e < 2 * NR; ++e) qs[w][e] = qa[c * STEPS + w][e];
          } else {
            const uint32_t addr = smem_u32(s_q + ((ROWS == 16 ? 0 : warp) * KSTEPS + c * STEPS + w) * 32 + lane);
            if constexpr (NR == 2) {
              const uint4 u = lds128(addr);
              qs[w][0] = u.x; qs[w][1] = u.y; qs[w][2] = u.z; qs[w][3] = u.w;
            } else {
              const uint2 u = lds64(addr);
              qs[w][0] = u.x; qs[w][1] = u.y;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < GROUPS; ++j) {
          const uint32_t at = kb + k_at[c % PIECES_BOX] + (c / PIECES_BOX) * (KEYS * TL::kRow) + 16 * j * TL::kRow;
          const uint4 us = lds128(at), vs = lds128(at + 8 * TL::kRow);
          const uint32_t u[4] = {us.x, us.y, us.z, us.w}, v[4] = {vs.x, vs.y, vs.z, vs.w};
#pragma unroll
          for (int i = 0; i < STEPS; ++i) {
            uint32_t x[4];
            if constexpr (F8) {
              x[0] = halves_of_codes(u[i]); x[1] = halves_of_codes(v[i]); x[2] = halves_of_codes(u[i] >> 16); x[3] = halves_of_codes(v[i] >> 16);
            } else {
              x[0] = u[2 * i]; x[1] = v[2 * i]; x[2] = u[2 * i + 1]; x[3] = v[2 * i + 1];
            }
#pragma unroll
            for (int r = 0; r < NR; ++r) mma<M>(CHAINS == 2 && i % 2 ? s_odd[0] : s[j][r], x[0], x[1], x[2], x[3], qs[i][r], qs[i][NR + r]);
          }
        }
      }
      if constexpr (CHAINS == 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[0][0][e] += s_odd[0][e];
      }
      // ---- running maxima --------------------------------------------------------------------------------------------------
      float mx[NR][2], mt[NR][2], lv[GROUPS];
#pragma unroll
      for (int r = 0; r < NR; ++r) mx[r][0] = mx[r][1] = mt[r][0] = mt[r][1] = -INFINITY;
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        float ks = 1.f;
        lv[j] = 0.f;
        if constexpr (F8) {
          const int at = a.P >= KEYS ? 0 : 16 * j >> page_bits;
          const float2 sc = s_scale[stage * 4 + at];
          ks = sc.y == sc.y ? sc.x : sc.y;                                   // a page whose values hold no numbers shows at the keys that are seen
          lv[j] = sc.y == sc.y ? sc.y : 0.f;
        }
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float f = by_row[r][e] * ks;
            float v = s[j][r][e] * f, w = s[j][r][2 + e] * f;
            if (masked) {
              const int key = key0 + 16 * j + pi, p = pos[r][e];
              if (key > p || (a.window > 0 && key <= p - a.window)) v = -INFINITY;
              if (key + 8 > p || (a.window > 0 && key + 8 <= p - a.window)) w = -INFINITY;
            }
            s[j][r][e] = v;
            s[j][r][2 + e] = w;
            const float top_j = fmaxf(v, w);
            mx[r][e] = fmaxf(mx[r][e], top_j);
            if (F8) mt[r][e] = fmaxf(mt[r][e], top_j + lv[j]);
          }
      }
      bool grew = false;
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          grew |= mx[r][e] > m[r][e];
          if (F8) grew |= mt[r][e] > top[r][e];
        }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
              mx[r][e] = fmaxf(mx[r][e], __shfl_xor_sync(0xffffffffu, mx[r][e], x));
              if (F8) mt[r][e] = fmaxf(mt[r][e], __shfl_xor_sync(0xffffffffu, mt[r][e], x));
            }
            const float m_new = fmaxf(m[r][e], mx[r][e]), t_new = F8 ? fmaxf(top[r][e], mt[r][e]) : m_new;
            l[r][e] *= m[r][e] == m_new ? 1.f : pt_exp2(m[r][e] - m_new);
            const float f = top[r][e] == t_new ? 1.f : pt_exp2(top[r][e] - t_new);
            m[r][e] = m_new;
            top[r][e] = t_new;
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
              o[i][r][e] *= f;
              o[i][r][2 + e] *= f;
            }
          }
      }
      // ---- probabilities, turned so that a lane holds row g's keys 2 t and 2 t + 1, and their product with the values ----------------
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        uint32_t pb[NR][2];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float ref = m[r][e] == -INFINITY ? 0.f : m[r][e];
            // 16-bit pages: no scales, top == m
            const float by = F8 ? (lv[j] == -INFINITY ? 0.f : pt_exp2(fminf(lv[j] + ref - top[r][e], 100.f) + kShift)) : (__is_same(M, __half) ? 256.f : 1.f);
            p[e] = pt_exp2(s[j][r][e] - ref);
            p[2 + e] = pt_exp2(s[j][r][2 + e] - ref);
            l[r][e] += p[e] + p[2 + e];
            p[e] *= by;
            p[2 + e] *= by;
          }
          pb[r][0] = transposed(Num<M>::pack(p[0], p[1]));
          pb[r][1] = transposed(Num<M>::pack(p[2], p[3]));
        }
        // what lies past the sequence's end may be no number, and nothing times that neither
        const int left = masked ? sh.s.len - (key0 + 16 * j) : 16;
        const uint32_t v0 = vb + v_at[0] + 16 * j * TL::kRow, v1 = vb + v_at[1] + 16 * j * TL::kRow;
        const auto times = [&](int tile_of, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
          for (int r = 0; r < NR; ++r) mma<M>(o[tile_of][r], a0, a1, a2, a3, pb[r][0], pb[r][1]);
        };
        // codes e of two words -> two halves
        const auto pair = [](uint32_t x, uint32_t y, int e) { return halves_of_codes(pt_prmt(x, y, (4 + e) << 4 | e)); };
        if constexpr (F8 && D == 64) {
          uint2 x = lds64(v0), y = lds64(v1), z = lds64(v0 + 8 * TL::kRow), u = lds64(v1 + 8 * TL::kRow);
          if (left < 16) {
            if (2 * t >= left) x = make_uint2(0u, 0u);
            if (((2 * t + 1) ^ 4) >= left) y = make_uint2(0u, 0u);
            if (2 * t + 8 >= left) z = make_uint2(0u, 0u);
            if (((2 * t + 1) ^ 4) + 8 >= left) u = make_uint2(0u, 0u);
          }
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            times(e / 2, pair(x.x, y.x, e), pair(x.x, y.x, e + 1), pair(z.x, u.x, e), pair(z.x, u.x, e + 1));
            times(2 + e / 2, pair(x.y, y.y, e), pair(x.y, y.y, e + 1), pair(z.y, u.y, e), pair(z.y, u.y, e + 1));
          }
        } else {
#pragma unroll
          for (int c = 0; c < TL::kBoxes; ++c) {
            const uint32_t at = c * KEYS * TL::kRow;
            uint4 xs = lds128(v0 + at), ys = lds128(v1 + at), zs = lds128(v0 + at + 8 * TL::kRow), us = lds128(v1 + at + 8 * TL::kRow);
            if (left < 16) {
              if (2 * t >= left) xs = make_uint4(0u, 0u, 0u, 0u);
              if (((2 * t + 1) ^ 4) >= left) ys = make_uint4(0u, 0u, 0u, 0u);
              if (2 * t + 8 >= left) zs = make_uint4(0u, 0u, 0u, 0u);
              if (((2 * t + 1) ^ 4) + 8 >= left) us = make_uint4(0u, 0u, 0u, 0u);
            }
            const uint32_t x[4] = {xs.x, xs.y, xs.z, xs.w}, y[4] = {ys.x, ys.y, ys.z, ys.w}, z[4] = {zs.x, zs.y, zs.z, zs.w}, u[4] = {us.x, us.y, us.z, us.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              if constexpr (F8) {
#pragma unroll
                for (int e = 0; e < 4; e += 2) times(c * 8 + 2 * w + e / 2, pair(x[w], y[w], e), pair(x[w], y[w], e + 1), pair(z[w], u[w], e), pair(z[w], u[w], e + 1));
              } else {
                times(c * 4 + w, pt_prmt(x[w], y[w], 0x5410), pt_prmt(x[w], y[w], 0x7632), pt_prmt(z[w], u[w], 0x5410), pt_prmt(z[w], u[w], 0x7632));
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + stage);
    }
    turn = first_turn + max(0, sh.last - sh.first);
    // ---- the piece's result: in units of 2^top where the keys have scales, l over the lanes of a row ----------------------------------
    constexpr float kUndo = __is_same(M, __half) ? 1.f / 256.f : 1.f;
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[r][e] += __shfl_xor_sync(0xffffffffu, l[r][e], x);
        if (!F8) top[r][e] = m[r][e];
      }
    const bool done = sh.begins && sh.ends;
    const int slot = first_piece ? 0 : 1, piece = 2 * blockIdx.x + slot;
    const long long first_row = sh.s.row;
    // channels 8 kRun c + kRun g + 4 q .. + 3 of row (r, e)
    const auto four = [&](int r, int e, int c, int q, float f) {
      const int k = c * (TL::kRun / 2) + 2 * q;
      return make_float4(o[k][r][e] * f, o[k][r][2 + e] * f, o[k + 1][r][e] * f, o[k + 1][r][2 + e] * f);
    };
    if constexpr (ROWS == 16) {
      // a thread has a row and a run of the box: the warps' factors once, then 32 channels at a time, four of each of a box's eight runs
      asm volatile("bar.sync 1, %0;" ::"n"(kSync) : "memory");              // the last piece's sums are no longer read
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (g == 0) *reinterpret_cast<float4*>(s_stats + (warp * 16 + 8 * r + 2 * t + e) * 4) = make_float4(m[r][e], l[r][e], top[r][e], 0.f);
      const int row_in = tid >> 3;
      float by_warp[kWarps], mm = -INFINITY, tt = -INFINITY, ll = 0.f, scale_out = kUndo;
      T* dst = nullptr;
      float* sums = nullptr;
#pragma unroll
      for (int part = 0; part < D / 32; ++part) {
        const int c = part / (TL::kRun / 4), q = part % (TL::kRun / 4);
        if (part > 0) asm volatile("bar.sync 1, %0;" ::"n"(kSync) : "memory");      // the last channels are no longer read
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e) *reinterpret_cast<float4*>(s_sum + (warp * 8 * NR + 8 * r + 2 * t + e) * 32 + 4 * g) = four(r, e, c, q, 1.f);
        asm volatile("bar.sync 1, %0;" ::"n"(kSync) : "memory");
        if (row_in >= used) continue;
        if (part == 0) {
          float4 st[kWarps];
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            st[w] = *reinterpret_cast<const float4*>(s_stats + (w * 16 + row_in) * 4);
            mm = fmaxf(mm, st[w].x);
            tt = fmaxf(tt, st[w].z);
          }
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            if (st[w].x != -INFINITY || st[w].y != 0.f) ll += st[w].y * (st[w].x == -INFINITY ? 1.f : pt_exp2(st[w].x - mm));
            by_warp[w] = st[w].z == -INFINITY ? (st[w].y != st[w].y ? 1.f : 0.f) : pt_exp2(st[w].z - tt);
          }
          if (done) {
            const int row = sh.row_tile * ROWS + row_in;
            scale_out = ll > 0.f || ll != ll ? kUndo * (F8 ? pt_exp2(tt - mm) : 1.f) / ll : 0.f;
            dst = static_cast<T*>(a.out) + ((first_row + row / R) * a.H + sh.head * R + row % R) * D;
          } else {
            sums = part_sums(a, gridDim.x, ROWS, piece) + static_cast<long long>(row_in) * D;
            if ((tid & 7) == 0) *reinterpret_cast<float4*>(part_stats(a, gridDim.x, ROWS, piece) + row_in * 4) = make_float4(mm, ll, tt, 0.f);
          }
        }
        const int d = (8 * c + (tid & 7)) * TL::kRun + 4 * q;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(s_sum + (w * 8 * NR + row_in) * 32 + 4 * (tid & 7));
          v.x += x.x * by_warp[w]; v.y += x.y * by_warp[w]; v.z += x.z * by_warp[w]; v.w += x.w * by_warp[w];
        }
        v = make_float4(v.x * scale_out, v.y * scale_out, v.z * scale_out, v.w * scale_out);
        if (done) write4(dst + d, v);
        else *reinterpret_cast<float4*>(sums + d) = v;
      }
    } else {
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int in_tile = warp_row + 8 * r + 2 * t + e, row = sh.row_tile * ROWS + in_tile;
          if (in_tile >= used) continue;
          const float ll = l[r][e], f = !done ? kUndo : ll > 0.f || ll != ll ? kUndo * (F8 ? pt_exp2(top[r][e] - m[r][e]) : 1.f) / ll : 0.f;
          T* dst = static_cast<T*>(a.out) + ((first_row + row / R) * a.H + sh.head * R + row % R) * D;
          float* sums = part_sums(a, gridDim.x, ROWS, piece) + static_cast<long long>(in_tile) * D;
#pragma unroll
          for (int c = 0; c < D / (8 * TL::kRun); ++c)
#pragma unroll
            for (int q = 0; q < TL::kRun / 4; ++q) {
              const int d = (8 * c + g) * TL::kRun + 4 * q;
              const float4 v = four(r, e, c, q, f);
              if (done) write4(dst + d, v);
              else *reinterpret_cast<float4*>(sums + d) = v;
            }
          if (!done && g == 0) *reinterpret_cast<float4*>(part_stats(a, gridDim.x, ROWS, piece) + in_tile * 4) = make_float4(m[r][e], ll, top[r][e], 0.f);
        }
    }
    if (sh.begins && !sh.ends) head = {sh.s.row, sh.head, used, static_cast<int>((sh.item_end - 1) / sh.per), slot, {sh.row_tile, 0, 0}};
    first_piece = false;
  }
  if (tid == 0 && !a.whole) *reinterpret_cast<PartHead*>(a.part + blockIdx.x * 8LL) = head;
  if constexpr (!F8) {
    __syncthreads();
    if (*met_odd != 0) add_odd<T, D, ROWS, KEYS>(a);
  }
}

// Joins the pieces of the item that begins in share blockIdx.x and goes on in the next ones; row by row over blockIdx.y, a lane for 4 channels, the pieces dealt
// out to the groups of lanes and added up in their order.
template <typename T, int ROWS>
__global__ void __launch_bounds__(128) paged_attention_join_kernel(const __grid_constant__ PagedAttnArgs a, int ctas) {
  pdl_entry();
  __shared__ float4 s_v[128];
  __shared__ float s_l[128];
  const PartHead h = *reinterpret_cast<const PartHead*>(a.part + blockIdx.x * 8LL);
  if (h.last < 0) return;
  const int lanes = a.D / 4, d = threadIdx.x % lanes * 4, group = threadIdx.x / lanes, groups = 128 / lanes, R = a.H / a.G;
  const int n = h.last - static_cast<int>(blockIdx.x) + 1;
  auto piece_of = [&](int i) { return i == 0 ? 2 * static_cast<int>(blockIdx.x) + h.slot : 2 * (static_cast<int>(blockIdx.x) + i); };
  for (int r = blockIdx.y; r < h.used; r += gridDim.y) {
    float m = -INFINITY, top = -INFINITY;
    for (int i = threadIdx.x & 31; i < n; i += 32) {
      const float4 st = *reinterpret_cast<const float4*>(part_stats(a, ctas, ROWS, piece_of(i)) + r * 4);
      m = fmaxf(m, st.x);
      top = fmaxf(top, st.z);
    }
    m = warp_max(m);
    top = warp_max(top);
    float l = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = group; i < n; i += groups) {
      const int piece = piece_of(i);
      const float4 st = *reinterpret_cast<const float4*>(part_stats(a, ctas, ROWS, piece) + r * 4);
      const float4 x = *reinterpret_cast<const float4*>(part_sums(a, ctas, ROWS, piece) + static_cast<long long>(r) * a.D + d);
      if (st.x != -INFINITY || st.y != 0.f) l += st.y * (st.x == -INFINITY ? 1.f : pt_exp2(st.x - m));
      const float f = st.z == -INFINITY ? (st.y != st.y ? 1.f : 0.f) : pt_exp2(st.z - top);
      v.x += x.x * f; v.y += x.y * f; v.z += x.z * f; v.w += x.w * f;
    }
    s_v[threadIdx.x] = v;
    s_l[threadIdx.x] = l;
    __syncthreads();
    if (group == 0) {
      for (int k = 1; k < groups; ++k) {
        const float4 x = s_v[k * lanes + threadIdx.x];
        v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
        l += s_l[k * lanes + threadIdx.x];
      }
      const int row = h.pad[0] * ROWS + r;
      const float f = l > 0.f || l != l ? pt_exp2(top - m) / l : 0.f;
      write4(static_cast<T*>(a.out) + ((h.row + static_cast<long long>(row / R)) * a.H + h.heads * R + row % R) * a.D + d, make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
    }
    __syncthreads();
  }
}

// The pages of every sequence as the ragged form of the attention kernel on tcgen05 (csrc/attention_fwd.cu) takes them: keys and values [B, G, capacity, D] in the
// queries' type, zeros behind the end up to a multiple of 128.  A (sequence, head) is one blockIdx.(z, y).  A page outside the cache,
// and the codes of one whose scales are no numbers, give keys that are none and values of zero, so that it shows at the rows that see it.  Rows of no sequence, or of one whose operands do not go together, are zeroed on the way.
// Values that are not finite go to a place of their own, with a flag for each warp's tokens, and are zeros among the values.
template <typename T, bool F8>
__global__ void __launch_bounds__(256) paged_gather_kernel(const __grid_constant__ PagedAttnArgs a, void* k_out, void* v_out, void* odd_out, uint8_t* odd_flags, long long capacity) {
  pdl_entry();
  const int b = blockIdx.z, head = blockIdx.y, lanes = a.D / 8, lane = threadIdx.x % lanes, per = 256 / lanes;
  if (head == 0) {
    const auto clear = [&](int row) {
      for (int i = threadIdx.x * 8; i < a.H * a.D; i += 2048) *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + static_cast<long long>(row) * a.H * a.D + i) = make_uint4(0u, 0u, 0u, 0u);
    };
    if (b == 0)
      for (int row = blockIdx.x; row < a.rows; row += gridDim.x)
        if (row < a.starts[0] || row >= a.starts[a.B]) clear(row);
    const Rows r = rows_of(a, b);
    if (!r.fits)
      for (int row = max(r.row, 0) + blockIdx.x; row < min(r.end, a.rows); row += gridDim.x) clear(row);
  }
  const Seq s = seq_of<16, 128>(a, b);
  if (s.n == 0) return;
  const int end = min(static_cast<long long>((s.len + 127) / 128 * 128), capacity), page_bits = 31 - __clz(a.P);
  // four tokens a thread, their pages and then their rows in flight together
  for (int token0 = s.tile0 * 128 + blockIdx.x * 4 * per; token0 < end; token0 += gridDim.x * 4 * per) {
    long long from[4];
    float ks[4], vs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int token = token0 + i * per + threadIdx.x / lanes;
      from[i] = -1;
      if (token >= s.len) continue;
      const int page = a.table[b * a.table_row + (token >> page_bits)];
      if (page < 0 || page >= a.pages) {                                    // outside the cache: nothing is read
        report_error(a.err, ERR_BOUNDS, page);
        from[i] = -2;
        continue;
      }
      const long long at = static_cast<long long>(page) * a.G + head;
      from[i] = (at * a.P + (token & (a.P - 1))) * a.D + lane * 8;
      if (F8) ks[i] = a.k_scale[at], vs[i] = a.v_scale[at];
    }
    typedef typename std::conditional<F8, uint2, uint4>::type Raw;          // eight channels
    Raw k[4], v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      k[i] = v[i] = Raw{};
      if (from[i] < 0) continue;
      k[i] = *reinterpret_cast<const Raw*>(static_cast<const uint8_t*>(a.k_pages) + from[i] * (F8 ? 1 : 2));
      v[i] = *reinterpret_cast<const Raw*>(static_cast<const uint8_t*>(a.v_pages) + from[i] * (F8 ? 1 : 2));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int token = token0 + i * per + threadIdx.x / lanes;
      if (token >= end) continue;
      const long long to = ((static_cast<long long>(b) * a.G + head) * capacity + token) * a.D + lane * 8;
      uint4 x, y;
      if constexpr (F8) {
        const bool none = from[i] < 0, lost = from[i] == -2 || (!none && vs[i] != vs[i]);
        const float kf = lost ? __uint_as_float(0x7fffffffu) : none ? 0.f : ks[i], vf = none || lost ? 0.f : vs[i];
        const auto two = [](uint32_t codes, float scale) {
          const float2 f = Num<__half>::two(halves_of_codes(codes));
          return Num<T>::pack(f.x * scale, f.y * scale);
        };
        x = make_uint4(two(k[i].x, kf), two(k[i].x >> 16, kf), two(k[i].y, kf), two(k[i].y >> 16, kf));
        y = make_uint4(two(v[i].x, vf), two(v[i].x >> 16, vf), two(v[i].y, vf), two(v[i].y >> 16, vf));
      } else {
        x = from[i] == -2 ? make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu) : k[i];
        y = v[i];
      }
      const uint4 all = y;
      const bool odd = __any_sync(0xffffffffu, without_odd<T>(y));          // a warp has whole tokens, all before `end`
      if (threadIdx.x % 32 == 0) odd_flags[to >> 8] = odd;
      if (odd) *reinterpret_cast<uint4*>(static_cast<T*>(odd_out) + to) = make_uint4(all.x ^ y.x, all.y ^ y.y, all.z ^ y.z, all.w ^ y.w);
      *reinterpret_cast<uint4*>(static_cast<T*>(k_out) + to) = x;
      *reinterpret_cast<uint4*>(static_cast<T*>(v_out) + to) = y;
    }
  }
}

typedef CUresult (*PagedEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Pages as the tiles want them: boxes of min(P, KEYS) tokens of one page and head, in columns of 128 bytes (a whole row where it is shorter).  A page outside the cache
// comes as zeros; keys in 16 bits as NaN (those in 8 have a scale for that).
template <typename T, bool F8, int D, int KEYS>
int page_map(CUtensorMap* map, const void* base, const PagedAttnArgs& a, bool keys) {
  static const PagedEncodeFn encode = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess
               ? reinterpret_cast<PagedEncodeFn>(ptr) : nullptr;
  }();
  if (encode == nullptr) return -20;
  using TL = Tile<F8, D, KEYS>;
  // [row of 128 bytes][token][128-byte column][page and head]; a page that is part of a tile comes column by column
  const cuuint32_t rows = a.P < KEYS ? a.P : KEYS, columns = a.P < KEYS ? 1 : TL::kBoxes;
  const cuuint64_t dims[4] = {TL::kRow / TL::kBytes, static_cast<cuuint64_t>(a.P), TL::kBoxes, static_cast<cuuint64_t>(a.pages) * a.G};
  const cuuint64_t strides[3] = {D * TL::kBytes, TL::kRow, static_cast<cuuint64_t>(a.P) * D * TL::kBytes};
  const cuuint32_t box[4] = {TL::kRow / TL::kBytes, rows, columns, 1}, step[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type = F8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : __is_same(T, __half) ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUresult r = encode(map, type, 4, const_cast<void*>(base), dims, strides, box, step,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, TL::kRow == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                            keys && !F8 ? CU_TENSOR_MAP_FLOAT_OOB_FILL_NAN_REQUEST_ZERO_FMA : CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 4000 + static_cast<int>(r);
}

// What to do with a form of the kernel: launch it, or say how many of its CTAs the device holds at once.
struct PagedCall {
  const PagedAttnArgs* a;
  cudaStream_t stream;
};

template <typename T, bool F8, int D, int ROWS, int NR>
int paged_form(const PagedCall& call) {
  constexpr int kSmem = Form<F8, D, ROWS, NR>::kSmem;
  const auto kernel = paged_attention_kernel<T, F8, D, ROWS, NR>;
  static OncePerDevice ready;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -32;
  if (ready(dev, [&] { return static_cast<int>(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem)); }) != 0) return -30;
  if (call.a == nullptr) {
    int per = 0, sms = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, Form<F8, D, ROWS, NR>::kThreads, kSmem) != cudaSuccess) return -31;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return -32;
    return per * sms;
  }
  const PagedAttnArgs& a = *call.a;
  CUtensorMap mk, mv;
  int r = page_map<T, F8, D, Form<F8, D, ROWS, NR>::kKeys>(&mk, a.k_pages, a, true);
  if (r == 0) r = page_map<T, F8, D, Form<F8, D, ROWS, NR>::kKeys>(&mv, a.v_pages, a, false);
  if (r != 0) return r;
  const int R = a.H / a.G;
  const long long items = (a.starts ? static_cast<long long>(a.rows) * R / ROWS + a.B : static_cast<long long>(a.B) * ((R + ROWS - 1) / ROWS)) * a.G;
  // whole items are dealt out evenly too
  const int n = a.whole ? static_cast<int>(items < 148 * 8 ? items : 148 * 8) : a.ctas;
  if (n <= 0) return -21;
  const cudaError_t e = launch_dependent(kernel, dim3(n), dim3(Form<F8, D, ROWS, NR>::kThreads), kSmem, call.stream, a, mk, mv);
  if (e != cudaSuccess || a.whole) return static_cast<int>(e);
  return static_cast<int>(launch_dependent(paged_attention_join_kernel<T, ROWS>, dim3(n, ROWS > 16 ? ROWS / 2 : a.starts ? 16 : (R < 16 ? R : 16)), dim3(128), 0, call.stream, a, n));
}

template <typename T, bool F8, int D>
int paged_rows(const PagedCall& call, int rows, bool few) {
  if (rows > 16) return paged_form<T, F8, D, D == 256 ? 64 : 128, 2>(call);
  return few ? paged_form<T, F8, D, 16, 1>(call) : paged_form<T, F8, D, 16, 2>(call);
}
template <typename T, bool F8>
int paged_dim(const PagedCall& call, int D, int rows, bool few) {
  switch (D) {
    case 64: return paged_rows<T, F8, 64>(call, rows, few);
    case 128: return paged_rows<T, F8, 128>(call, rows, few);
    case 256: return paged_rows<T, F8, 256>(call, rows, few);
  }
  return -2;
}
int paged_type(const PagedCall& call, int dtype, bool f8, int D, int rows, bool few) {
  if (rows != 16 && rows != (D == 256 ? 64 : 128)) return -3;
  if (dtype == 0) return f8 ? paged_dim<__nv_bfloat16, true>(call, D, rows, few) : paged_dim<__nv_bfloat16, false>(call, D, rows, few);
  if (dtype == 1) return f8 ? paged_dim<__half, true>(call, D, rows, few) : paged_dim<__half, false>(call, D, rows, few);
  return -6;
}

}  // namespace tyr

int tyr_flash_fwd_ragged(const void* q, long long q_row, long long q_head, const void* k, const void* v, const void* odd, const uint8_t* odd_flags, void* out, const int* starts, const int* lengths, int rows, int B,
                         int Hq, int Hkv, int D, long long capacity, int longest, int window, float scale, int dtype, int* err, cudaStream_t stream);

using namespace tyr;

// The same result for many new tokens a sequence: the pages laid out in `part` (with n = B * G * capacity * D: n keys, n values and room for n values that are not
// finite, in the queries' type, and n / 256 bytes of flags; capacity a multiple of 128 that holds the table's tokens), then the kernel on tcgen05.
extern "C" TYR_EXPORT int tyr_paged_attention_gathered(const void* packed, int dtype, long long capacity, void* stream) {
  const PagedAttnArgs& a = *static_cast<const PagedAttnArgs*>(packed);
  if (a.rows <= 0 || a.B <= 0 || a.B > 65535 || a.H <= 0 || a.G <= 0 || a.G > 65535 || a.H % a.G != 0 || a.pages <= 0 || a.width <= 0 || a.window < 0) return -1;
  if ((a.P != 16 && a.P != 32 && a.P != 64 && a.P != 128) || (a.D != 64 && a.D != 128) || a.starts == nullptr || a.part == nullptr) return -2;
  if (capacity % 128 != 0 || capacity < static_cast<long long>(a.width) * a.P || capacity > 0x7fffffffLL || (a.k_scale != nullptr) != (a.v_scale != nullptr)) return -3;
  const long long numbers = static_cast<long long>(a.B) * a.G * capacity * a.D;
  uint8_t* work = reinterpret_cast<uint8_t*>(a.part);
  void *k = work, *v = work + 2 * numbers, *odd = work + 4 * numbers;
  uint8_t* flags = work + 6 * numbers;
  // some eight rounds of blocks over the SMs' places, or as many as the longest sequence may fill
  const long long chunks = capacity * a.D / 8192, most = 9472 / (static_cast<long long>(a.G) * a.B) + 1;
  const dim3 grid(static_cast<unsigned>(chunks < most ? chunks : most), a.G, a.B);
  const bool f8 = a.k_scale != nullptr;
  const auto gather = dtype == 0 ? (f8 ? paged_gather_kernel<__nv_bfloat16, true> : paged_gather_kernel<__nv_bfloat16, false>)
                                 : (f8 ? paged_gather_kernel<__half, true> : paged_gather_kernel<__half, false>);
  const cudaError_t e = launch_dependent(gather, grid, dim3(256), 0, (cudaStream_t)stream, a, k, v, odd, flags, capacity);
  if (e != cudaSuccess) return static_cast<int>(e);
  return tyr_flash_fwd_ragged(a.q, a.q_row, a.q_head, k, v, odd, flags, a.out, a.starts, a.lengths, a.rows, a.B, a.H, a.G, a.D, capacity, a.width * a.P, a.window, a.scale, dtype, a.err, (cudaStream_t)stream);
}

// dtype: 0 = bf16, 1 = fp16 (queries, results, and pages without scales); rows of a tile: 16, or 128 (64 of heads of 256).
extern "C" TYR_EXPORT int tyr_paged_attention(const void* packed, int dtype, int rows, void* stream) {
  const PagedAttnArgs& a = *static_cast<const PagedAttnArgs*>(packed);
  if (a.rows <= 0 || a.B <= 0 || a.H <= 0 || a.G <= 0 || a.H % a.G != 0 || a.pages <= 0 || a.width <= 0 || a.window < 0) return -1;
  if (a.P != 16 && a.P != 32 && a.P != 64 && a.P != 128) return -2;
  if ((a.k_scale != nullptr) != (a.v_scale != nullptr) || (!a.whole && (a.part == nullptr || a.ctas <= 0))) return -3;
  // a sequence's work and the pages' rows are counted in 32 bits
  const int keys = tile_keys(rows, a.D * (a.k_scale ? 1 : 2));
  const long long tiles = (static_cast<long long>(a.width) * a.P + keys - 1) / keys;
  if ((static_cast<long long>(a.rows) * (a.H / a.G) / rows + 1) * a.G * tiles > 0x7fffffffLL || static_cast<long long>(a.pages) * a.G > 0x7fffffffLL) return -4;
  if (static_cast<long long>(a.width) * a.P > 0x7fffffffLL || static_cast<long long>(a.rows) * a.H > 0x7fffffffLL) return -5;
  return paged_type(PagedCall{&a, (cudaStream_t)stream}, dtype, a.k_scale != nullptr, a.D, rows, a.starts == nullptr && a.H / a.G <= 8);
}

// CTAs of a form that the current device holds at once (few: at most 8 rows in a tile of 16); negative: an error.
extern "C" TYR_EXPORT int tyr_paged_attention_resident(int dtype, int f8, int D, int rows, int few) {
  return paged_type(PagedCall{nullptr, nullptr}, dtype, f8 != 0, D, rows, few != 0);
}
