// Attention of new tokens over a paged KV cache: decode steps and a few drafted tokens
// (bf16 or 4-bit pages; bf16 queries and outputs, fp32 scores, softmax and accumulation).
//
// Columns n = i group + h of a KV head (token i of T, query head h of the group) share its K
// and V; 16 of them are one tile. A stream is a (sequence, KV head, column tile), its work
// ceil(keys / unit) units.
//
// Bound: HBM (each visible row of K and V once per column tile); with 4-bit pages the unpacking
// is close behind (some 120 vector instructions per 16 keys); with one unit per workgroup the chain
// lengths -> page ids -> K and V -> merge (bf16 pages: lengths -> Q -> page ids, whose load the
// compiler moves behind the wait for Q). Measured, main kernel + merge: 8 ragged sequences of up to
// 16000 keys (32/8 heads, bf16) 50 + 4.8 us, the 314 MB at 5.7 TB/s; 64 of up to 8192 in 4 bits
// 71 + 4.8, 301 MB at 4.0 TB/s; 131072 keys (28/4, 4 bits) 20 + 4.0; 32641 keys 8.3 + 3.7; 1090 keys
// in bf16 6.0 + 3.7.
//   * The streams' units, in order, are dealt in equal runs to the workgroups of one grid that
//     fills the chip. The lengths are device data, so every workgroup finds its run itself:
//     a prefix sum over the batch in one wave (a load and some shuffles), no host
//     synchronisation, and a captured launch can be replayed with other lengths. A stream
//     that falls to one workgroup is written out directly; of the others each workgroup
//     leaves at most two partial results (its run's first and last stream), joined by a
//     second kernel in a fixed order.
//   * A unit is a few 16-key tiles per wave, four waves. Page ids come from a register that holds
//     those of the wave's next 64 tiles, so no load waits for a page table entry of its own.
//   * Scores: S^T = K Q^T, v_mfma_f32_16x16x32_bf16, K rows as A operand straight from memory.
//     The order of the dims in the sum is free: with 4-bit pages a lane takes 32 consecutive
//     dims of a row, which are 16 bytes and one scale, widened exactly to bf16 by
//     v_cvt_scalef32_pk_bf16_fp4 (two values and their scale an instruction).
//   * P V: v_mfma_f32_16x16x32_bf16 over the keys of two tiles. Their scores lie in the lane as
//     the A operand wants them; a lane holds its dims of the eight rows it needs, and byte
//     permutes pair the keys. P goes through in three bf16 parts, 24 bits as in fp32, and its sums
//     are products of the same parts with ones: products and LSE are those of an fp32 P. (Two parts
//     lose up to 2^-17, and an LSE is off by as much, which no rounding of the output covers. The third
//     costs 2 to 6 % with 4-bit pages, 64 sequences of 8192 keys 114 -> 121 us, 131072 keys 25.3 ->
//     26.8, and nothing with bf16 pages.) Where that makes NaN (infinite values of bf16 pages meet a
//     part of P that is 0) the wave runs again with P as it is, v_mfma_f32_16x16x4_f32.
//   * The running maximum is raised, and O scaled, only in steps where it grows.
#include <algorithm>
#include <cmath>

#include "paged_tiles.h"

namespace spx {

constexpr int kPaCols = 16;
constexpr int kPaMaxGrid = 1024;         // workgroups that share the units (weights in the merge)
constexpr int kPaCus = 256;
constexpr int kPaMinUnit = 128;          // keys of the smallest unit

// W waves per workgroup.
template <int D, bool kFour, int W>
struct PagedShape {
  static constexpr int kTiles = kFour && D == 128 ? 4 : 2;     // of a wave and unit
  static constexpr int kUnit = 16 * kTiles * W;                // keys of a unit
  static_assert(kUnit >= kPaMinUnit, "units are counted in 32 bits");
  static constexpr int kPerCu = W == 8 ? 1 : 2;                // resident workgroups
  static constexpr bool kEarlyKeys = kFour || D == 128;        // registers for them
};

struct PagedAttnArgs {
  PagedMap map;
  const uint16_t* q;
  int64_t qs_b, qs_t, qs_h;
  const void* key_pages;
  const void* value_pages;
  const uint8_t* key_scales;
  const uint8_t* value_scales;
  int batch, tokens, q_heads, kv_heads, group;
  int cols, col_tiles;                   // tokens x group, tiles of 16 of them
  int grid;                              // workgroups sharing the units; 0: one per stream
  double inv_grid, inv_group;            // reciprocals
  float scale_log2;                      // > 0: the sign of the scale, or a scale of 0, goes to q
  uint32_t q_keep, q_flip;               // q & q_keep ^ q_flip
  uint16_t* out;
  float* lse;
  float* part_o;                         // [2 grid][16][D]
  float* part_ml;                        // [2 grid][16][2]
  u32x2* parts;                          // [streams] first partial's slot, how many (1: written out)
};

// Weight of a partial with maximum m in a merge with maximum top: an empty partial
// (m = -inf) counts nothing, also where every partial is empty.
__device__ __forceinline__ float part_weight(float m, float top) {
  return m == -INFINITY ? 0.0f : exp2_fast(m - top);
}

// ---------------------------------------------------------------- division of the work

// Live tokens of a sequence: 0 .. live - 1.
__device__ __forceinline__ int live_tokens(const PagedAttnArgs& a, int start, int count) {
  const int64_t room = a.map.capacity() - start;
  const int live = min(min(count, a.tokens), (int)min(room, (int64_t)a.tokens));
  return start < 0 ? 0 : max(live, 0);
}

// Tokens of a column tile: the first and the last.
__device__ __forceinline__ int tile_first(const PagedAttnArgs& a, int tile) {
  return a.col_tiles == 1 ? 0 : divide(tile * kPaCols, a.group, a.inv_group);
}
__device__ __forceinline__ int tile_last(const PagedAttnArgs& a, int tile) {
  return a.col_tiles == 1
             ? a.tokens - 1
             : divide(min((tile + 1) * kPaCols, a.cols) - 1, a.group, a.inv_group);
}

__device__ __forceinline__ int column_token(const PagedAttnArgs& a, int column) {
  return a.tokens == 1 ? 0 : divide(column, a.group, a.inv_group);
}

// Keys that a column tile of a sequence sees at most.
__device__ __forceinline__ int tile_keys(const PagedAttnArgs& a, int start, int live, int tile) {
  const int last = min(tile_last(a, tile), live - 1);
  return last < tile_first(a, tile) ? 0 : start + last + 1;
}

// Units of a sequence's streams of one KV head.
template <int kUnit>
__device__ __forceinline__ int head_units(const PagedAttnArgs& a, int start, int live) {
  int units = 0;
  for (int tile = 0; tile < a.col_tiles; ++tile)
    units += (tile_keys(a, start, live, tile) + kUnit - 1) / kUnit;
  return units;
}

// The units of 64 sequences, one a lane, and their prefix sums.
struct UnitScan {
  int start, live, each, units, sum;     // each: of one KV head
  template <int kUnit>
  __device__ __forceinline__ void load(const PagedAttnArgs& a, int b) {
    start = -1;
    int count = a.tokens;
    if (b < a.batch) {
      start = a.map.starts[b];
      if (a.map.counts) count = a.map.counts[b];
    }
    live = live_tokens(a, start, count);
    each = head_units<kUnit>(a, start, live);
    units = each * a.kv_heads;
    sum = wave_prefix(units);
  }
  __device__ __forceinline__ int total() const { return __builtin_amdgcn_readlane(sum, kWave - 1); }
};

struct Run {                             // units begin(w) .. begin(w + 1) - 1 of workgroup w
  int per, rest;
  __device__ __forceinline__ Run(int total, int grid, double inv)
      : per(first_lane(divide(total, grid, inv))), rest(total - per * grid) {}
  __device__ __forceinline__ int begin(int w) const { return w * per + min(w, rest); }
  __device__ __forceinline__ int owner(int u) const {
    const int wide = rest * (per + 1);
    return u < wide ? u / (per + 1) : rest + (u - wide) / max(per, 1);
  }
};

struct Stream {
  int b, kvh, tile, start, live, keys, units;
  int first;                             // of its units

  __device__ __forceinline__ void lengths(const PagedAttnArgs& a) {
    start = scalar_load(a.map.starts + b);
    live = live_tokens(a, start, a.map.counts ? scalar_load(a.map.counts + b) : a.tokens);
  }
  template <int kUnit>
  __device__ __forceinline__ void measure(const PagedAttnArgs& a) {
    keys = tile_keys(a, start, live, tile);
    units = (keys + kUnit - 1) / kUnit;
  }
  // The stream of unit u; scan: that of the sequences 0 .. 63. false: there is none (lengths
  // that change under the launch must not make it loop).
  template <int kUnit>
  __device__ __forceinline__ bool find(const PagedAttnArgs& a, int lane, UnitScan scan, int u) {
    int before = 0, b0 = 0;
    uint64_t past;
    while (!(past = __ballot(before + scan.sum > u))) {
      before += scan.total();
      b0 += kWave;
      if (b0 >= a.batch) return false;
      scan.load<kUnit>(a, b0 + lane);
    }
    const int l = __builtin_ctzll(past);
    b = b0 + l;
    before += __builtin_amdgcn_readlane(scan.sum - scan.units, l);
    const int each = __builtin_amdgcn_readlane(scan.each, l);
    start = __builtin_amdgcn_readlane(scan.start, l);
    live = __builtin_amdgcn_readlane(scan.live, l);
    // fewer heads than fp32 has bits for
    kvh = first_lane((int)((float)(u - before) * __builtin_amdgcn_rcpf((float)each)));
    while (kvh * each > u - before) --kvh;
    while ((kvh + 1) * each <= u - before) ++kvh;
    first = before + kvh * each;
    for (tile = 0; tile < a.col_tiles; ++tile) {
      measure<kUnit>(a);
      if (u < first + units) return true;
      first += units;
    }
    return false;
  }
  // The next one that has units.
  template <int kUnit>
  __device__ __forceinline__ bool next(const PagedAttnArgs& a) {
    first += units;
    do {
      if (++tile == a.col_tiles) {
        tile = 0;
        if (++kvh == a.kv_heads) {
          kvh = 0;
          if (++b == a.batch) return false;
          lengths(a);
        }
      }
      measure<kUnit>(a);
    } while (units == 0);
    return true;
  }
};

// ------------------------------------------------------------------------- one stream

// The kernel arguments, read afresh: nothing derived from them is held across the loop over a
// stream's units (held, they cost its scalar registers, and spills to vector lanes inside the loop).
// What is left is kept outside it, stored before and read behind a stream: 19 to 23 scalar registers
// in vector lanes (4 bits, D = 128), 4 or 5 vector registers in scratch (bf16, D = 256).
__device__ __forceinline__ PagedAttnArgs fresh_args() {
#if defined(__HIP_DEVICE_COMPILE__)
  auto p = (const __attribute__((address_space(4))) PagedAttnArgs*)
      __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *p;
#else
  return {};
#endif
}

// All cache lines of the arguments at once: read where they are used, each line would be a
// wait of its own.
__device__ __forceinline__ void touch_args() {
#if defined(__HIP_DEVICE_COMPILE__)
  auto p = (const __attribute__((address_space(4))) int*)__builtin_amdgcn_kernarg_segment_ptr();
  int any = 0;
#pragma unroll
  for (size_t i = 0; i < sizeof(PagedAttnArgs); i += 64) any |= p[i / 4];
  asm volatile("" ::"s"(any));
#endif
}

__device__ __forceinline__ uint32_t opaque_bits(uint32_t x) { return (uint32_t)opaque((int)x); }

// The lane, recomputed where it is used: what rare paths derive from it is not held meanwhile.
__device__ __forceinline__ int thread_lane() { return opaque((int)threadIdx.x) & 63; }

__device__ __forceinline__ float sum_of_halves(float x) {
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

// Maximum over the lanes c, c + 16, c + 32, c + 48.
__device__ __forceinline__ float max_over_rows(float x) {
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
  const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}

// Dims of the lane c in a V row and an O register: D / 16 consecutive ones.
template <int D>
__device__ __forceinline__ int value_dim(int c, int i) {
  return D / 16 * c + i;
}

// Partial results keep the lanes' groups of four dims side by side (in the order of the dims, 16
// bytes every D / 4 from lane to lane, writing them to LDS met its banks four times): at `place`
// (a multiple of 4) are the dims from here on.
template <int D>
__device__ __forceinline__ int place_of(int c, int i) {
  return 4 * (16 * (i / 4) + c);
}
template <int D>
__device__ __forceinline__ int dim_at(int place) {
  return value_dim<D>(place / 4 % 16, place / 64 * 4);
}

template <int D, bool kFour>
struct ValueTile {                       // a lane's dims of four rows of V: 4 g + r
  static constexpr int kWords = kFour ? D / 128 : D / 32;
  uint32_t raw[4][kWords];
  uint32_t scale[kFour ? 4 : 1];         // four scale bytes of each row

  // The lane's byte of them.
  static __device__ __forceinline__ int scale_byte(int c) { return c * (D / 16) / kPagedGroup % 4; }

  __device__ __forceinline__ void load_row(GlobalBytes p, GlobalBytes s, int r, int at, int c) {
    if constexpr (kFour) {
      if constexpr (D == 128) {
        raw[r][0] = global_load<uint32_t>(p, at * 64 + 4 * c);
      } else {
        const u32x2 w = global_load<u32x2>(p, at * 128 + 8 * c);
        raw[r][0] = w[0];
        raw[r][1] = w[1];
        scale[r] = global_load<uint32_t>(s, at * 8 + 4 * (c / 8));
      }
    } else {
#pragma unroll
      for (int x = 0; x < D / 128; ++x) {
        const u32x4 w = global_load<u32x4>(p, at * 2 * D + D / 8 * c + 16 * x);
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[r][4 * x + e] = w[e];
      }
    }
  }
  __device__ __forceinline__ void load(const HeadPages<D, kFour>& h, int64_t row, int c, int g) {
    const GlobalBytes p = tile_base(h.values + row * h.kRowBytes);
    GlobalBytes s = p;
    if constexpr (kFour) s = tile_base(h.value_scales + row * h.kRowScales);
#pragma unroll
    for (int r = 0; r < 4; ++r) load_row(p, s, r, 4 * g + r, c);
    if constexpr (kFour && D == 128) {   // of the four rows: 16 bytes
      const u32x4 w = global_load<u32x4>(s, 16 * g);
#pragma unroll
      for (int r = 0; r < 4; ++r) scale[r] = w[r];
    }
  }
  __device__ __forceinline__ void clear(int r) {
#pragma unroll
    for (auto& x : raw[r]) x = 0;
    if constexpr (kFour) scale[r] = 0x7f7f7f7fu;
  }
  __device__ __forceinline__ bool finite(int r, int c) const {
    if constexpr (kFour) return (scale[r] >> (8 * scale_byte(c)) & 255) != 255;
    bool ok = true;
#pragma unroll
    for (uint32_t x : raw[r])
      ok = ok && (x & 0x7f80u) != 0x7f80u && (x & 0x7f800000u) != 0x7f800000u;
    return ok;
  }
  // Dims 2 x and 2 x + 1 of the lane's in row r as a bf16 pair.
  __device__ __forceinline__ uint32_t pair(int r, int x, int c) const {
    if constexpr (kFour) {
      const float size = scale_of(scale[r], scale_byte(c));
      const uint32_t w = raw[r][x / 4];
      return __builtin_bit_cast(
          uint32_t, x % 4 == 0   ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, size, 0)
                    : x % 4 == 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, size, 1)
                    : x % 4 == 2 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, size, 2)
                                 : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, size, 3));
    } else {
      return raw[r][x];
    }
  }
};

// What a wave needs of its stream in the loop over the units.
struct Limits {
  int b, keys;                           // the sequence, keys that any column sees
  int first;                             // the last key that the tile's first column sees
  int column;                            // and the one that column c sees
};

// A wave's tiles of a stream: page ids, keys and values of one unit, O and the softmax state.
// kHalf (4-bit pages): at most eight columns; column c + 8 is column c again, and holds the second
// part of its P in the products with V (the halves of O are added in the end): two of these
// instead of three.
template <int D, bool kFour, int W, bool kHalf>
struct Wave {
  using Shape = PagedShape<D, kFour, W>;
  using Pages = HeadPages<D, kFour>;
  static constexpr int T = Shape::kTiles, KK = D / 32, N = D / 16;
  static constexpr int kParts = kHalf ? 2 : 3;             // operands that hold P
  KeyTile<D, kFour> key[T];
  ValueTile<D, kFour> value[T];
  f32x4 o[N];                            // [query row 4 g + r][value_dim(c, i)]
  f32x4 l;                               // sums of P, query row 4 g + r
  float m;                               // maximum of column c, unscaled
  int ids, id_base;                      // lane i: page of tile i % T in unit id_base + i / T
  uint32_t bad;                          // tiles without a place

  __device__ __forceinline__ void load_ids(const Limits& s, int j, int w, int lane) {
    const PagedAttnArgs a = fresh_args();
    id_base = j;
    const int p = (j + lane / T) * Shape::kUnit + (w * T + lane % T) * 16;
    ids = a.map.page(s.b, min(p, s.keys - 1));
  }
  __device__ __forceinline__ int page(int j, int t) const {
    return __builtin_amdgcn_readlane(ids, (j - id_base) * T + t);
  }
  // Tiles without a place read page 0.
  __device__ __forceinline__ void load_keys(const Pages& h, int j, int key0, int c, int g) {
    bad = 0;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const int id = page(j, t);
      bad |= (id < 0 ? 1u : 0u) << t;
      key[t].load(h, h.row(max(id, 0), key0 + 16 * t), c, g);
    }
  }
  __device__ __forceinline__ void load_values(const Pages& h, int j, int key0, int c, int g) {
#pragma unroll
    for (int t = 0; t < T; ++t)
      value[t].load(h, h.row(max(page(j, t), 0), key0 + 16 * t), c, g);
  }

  // Units j .. end - 1; load_ids(s, j, w, lane) is done. The next unit's keys are fetched as soon
  // as the scores are formed, its values after the products. kWide: P V in fp32 products.
  template <bool kWide>
  __device__ __forceinline__ void run(const Pages& h, const Limits& s, const u32x4 (&q)[KK],
                                      float scale, int j, int end, int w, int lane, int c, int g) {
#pragma unroll
    for (auto& x : o) x = f32x4{};
    l = f32x4{};
    m = -INFINITY;
    const int offset = w * T * 16;       // the wave's first key in a unit
    end = min(end, (s.keys - offset + Shape::kUnit - 1) / Shape::kUnit);
    if (j >= end) return;
    load_keys(h, j, j * Shape::kUnit + offset, c, g);
    load_values(h, j, j * Shape::kUnit + offset, c, g);
    bool first = true;
    for (;;) {
      const int key0 = j * Shape::kUnit + offset;
      const bool more = j + 1 < end;
      const uint32_t unplaced = bad;
      f32x4 x[T];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < T; ++t) x[t] = f32x4{};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int t = 0; t < T; ++t) x[t] = mfma16(key[t].operand(kk, g), q[kk], x[t]);
      __builtin_amdgcn_sched_barrier(0);
      if (Shape::kEarlyKeys && more) {
        if (j + 1 - id_base >= kWave / T) load_ids(s, j + 1, w, lane);
        load_keys(h, j + 1, key0 + Shape::kUnit, c, g);
      }
      __builtin_amdgcn_sched_barrier(0);
      softmax_products<kWide>(h, s, x, scale, key0, unplaced, first, c, g);
      first = false;
      if (!more) return;
      ++j;
      __builtin_amdgcn_sched_barrier(0);
      if (!Shape::kEarlyKeys) {
        if (j - id_base >= kWave / T) load_ids(s, j, w, lane);
        load_keys(h, j, key0 + Shape::kUnit, c, g);
      }
      load_values(h, j, key0 + Shape::kUnit, c, g);
    }
  }

  template <bool kWide>
  __device__ __forceinline__ void softmax_products(const Pages& h, const Limits& s, f32x4 (&x)[T],
                                                   float scale, int key0, uint32_t unplaced,
                                                   bool first, int c, int g) {
    bool split = false;                  // V rows of some columns only, not finite: left out
    if (unplaced != 0 || key0 + 16 * T - 1 > s.first) {
      const int g = thread_lane() >> 4, c = thread_lane() & 15;
      // scores of keys that a column does not see are -inf; rows that no column sees are 0, so
      // that what lies behind the last token does not meet a probability of 0
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int p = key0 + 16 * t + 4 * g + r;
          const bool here = !(unplaced >> t & 1);
          if (!here || p > s.column) x[t][r] = -INFINITY;
          if (!here || p >= s.keys) {
            value[t].clear(r);
          } else if (p > s.first && !value[t].finite(r, c)) {
            split = true;
            value[t].clear(r);
          }
        }
    }
    float mx = x[0][0];
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, x[t][r]);
    mx = max_over_rows(mx);
    if (first) {
      m = mx;
    } else if (__any(mx > m)) {
      const float m_new = fmaxf(m, mx);
      const float corr = m == -INFINITY ? 0.0f : exp2_fast((m - m_new) * scale);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float cr = __shfl(corr, 4 * (thread_lane() >> 4) + r);
        l[r] *= cr;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i][r] *= cr;
      }
      m = m_new;
    }
    const float shift = m == -INFINITY ? 0.0f : m * scale;
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) x[t][r] = exp2_fast(__builtin_fmaf(x[t][r], scale, -shift));
    if constexpr (kWide) {
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          l = __builtin_amdgcn_mfma_f32_16x16x4f32(x[t][r], 1.0f, l, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < N; i += 2) {
            const uint32_t v2 = value[t].raw[r][i / 2];
            o[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[t][r], bf16_lo(v2), o[i], 0, 0, 0);
            o[i + 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[t][r], bf16_hi(v2), o[i + 1], 0, 0, 0);
          }
        }
    } else {
#pragma unroll
      for (int t = 0; t < T; t += 2) {
        // Three bf16 parts hold the 24 bits of an fp32 probability. kHalf: the first of column c and
        // the second of column c + 8 are one operand, the third and zeros the other.
        u32x4 part[kParts];
        const uint32_t upper = c < kPaCols / 2 ? 0 : ~0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float u = x[t + e / 2][2 * (e % 2)], w = x[t + e / 2][2 * (e % 2) + 1];
          const uint32_t p1 = opaque_bits(pack_bf16x2(u, w));
          u -= bf16_lo(p1);
          w -= bf16_hi(p1);
          const uint32_t p2 = opaque_bits(pack_bf16x2(u, w));
          const uint32_t p3 = pack_bf16x2(u - bf16_lo(p2), w - bf16_hi(p2));
          if constexpr (kHalf) {
            part[0][e] = (p1 & ~upper) | (p2 & upper);
            part[1][e] = p3 & ~upper;
          } else {
            part[0][e] = p1;
            part[1][e] = p2;
            part[2][e] = p3;
          }
        }
        const uint32_t ones = 0x3f803f80u;
#pragma unroll
        for (const auto& p : part) l = mfma16(p, u32x4{ones, ones, ones, ones}, l);
#pragma unroll
        for (int y = 0; y < N / 2; ++y) {
          uint32_t row[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) row[j] = value[t + j / 4].pair(j % 4, y, c);
          u32x4 even, odd;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            even[e] = __builtin_amdgcn_perm(row[2 * e + 1], row[2 * e], 0x05040100u);
            odd[e] = __builtin_amdgcn_perm(row[2 * e + 1], row[2 * e], 0x07060302u);
          }
#pragma unroll
          for (const auto& p : part) {
            o[2 * y] = mfma16(p, even, o[2 * y]);
            o[2 * y + 1] = mfma16(p, odd, o[2 * y + 1]);
          }
        }
      }
    }
    if (__any(split)) add_split_rows(h, s, x, key0);
  }

  // The V rows that were left out, one after the other: only into the columns that see them.
  __device__ __forceinline__ void add_split_rows(const Pages& h, const Limits& s,
                                                 const f32x4 (&p)[T], int key0) {
    const PagedAttnArgs a = fresh_args();
    const int g = thread_lane() >> 4, c = thread_lane() & 15;
    const int last = min(key0 + 16 * T, s.keys);
#pragma unroll 1
    for (int at = max(key0, s.first + 1); at < last; ++at) {
      const int id = a.map.page(s.b, at);
      if (id < 0) continue;
      const int64_t row = h.row(id, at);
      ValueTile<D, kFour> v;             // its row 0
      const GlobalBytes scales = kFour ? h.value_scales + row * h.kRowScales : h.values;
      v.load_row(h.values + row * h.kRowBytes, scales, 0, 0, c);
      if constexpr (kFour && D == 128) v.scale[0] = global_load<uint32_t>(scales, 0);
      const bool left_out = !v.finite(0, c);
      float mine = 0.0f;                 // the probability of key `at`, where this lane has it
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) mine = key0 + 16 * t + 4 * g + r == at ? p[t][r] : mine;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float prob = __shfl(mine, 16 * (at / 4 % 4) + 4 * g + r);
        const int seen = __shfl(s.column, 4 * g + r);
        const bool sees = left_out && at <= seen && (!kHalf || 4 * g + r < kPaCols / 2);
#pragma unroll
        for (int y = 0; y < N / 2; ++y) {
          const uint32_t w = v.pair(0, y, c);
          o[2 * y][r] += sees ? prob * bf16_lo(w) : 0.0f;
          o[2 * y + 1][r] += sees ? prob * bf16_hi(w) : 0.0f;
        }
      }
    }
  }

  // kHalf: rows 8 to 15 of O and the sums added to rows 0 to 7 (lanes 32 apart).
  __device__ __forceinline__ void add_halves() {
#pragma unroll
    for (auto& x : o)
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = sum_of_halves(x[r]);
#pragma unroll
    for (int r = 0; r < 4; ++r) l[r] = sum_of_halves(l[r]);
  }

  __device__ __forceinline__ bool any_nan() const {
    float sum = 0.0f;
#pragma unroll
    for (const auto& x : o)
#pragma unroll
      for (int r = 0; r < 4; ++r) sum = __builtin_fmaf(x[r], 0.0f, sum);
    return __any(sum != sum);
  }
};

// grid > 0: workgroup w takes its run of all units; grid == 0: workgroup w is stream w.
template <int D, bool kFour, int W, bool kHalf>
__global__ __launch_bounds__(64 * W, (PagedShape<D, kFour, W>::kPerCu * W / 4)) void
paged_attn_kernel(PagedAttnArgs args) {
  using Shape = PagedShape<D, kFour, W>;
  constexpr int KK = D / 32;
  __shared__ float part_m[W][kPaCols], part_l[W][kPaCols];
  __shared__ __align__(16) float part_o[W][kHalf ? kPaCols / 2 : kPaCols][D];
  const int lane = threadIdx.x & 63, w = first_lane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  touch_args();

  Stream s;
  Run run(0, 1, 1.0);
  int u, end;
  if (args.grid > 0) {
    UnitScan scan;
    scan.load<Shape::kUnit>(args, lane);
    int total = scan.total();
    for (int b0 = kWave; b0 < args.batch; b0 += kWave) {
      UnitScan more;
      more.load<Shape::kUnit>(args, b0 + lane);
      total += more.total();
    }
    run = Run(total, args.grid, args.inv_grid);
    u = run.begin(blockIdx.x);
    end = run.begin(blockIdx.x + 1);
    if (u >= end || !s.find<Shape::kUnit>(args, lane, scan, u)) return;
  } else {
    const int stream = blockIdx.x;
    s.tile = stream % args.col_tiles;
    s.kvh = stream / args.col_tiles % args.kv_heads;
    s.b = stream / args.col_tiles / args.kv_heads;
    s.first = u = 0;
    s.lengths(args);
    s.measure<Shape::kUnit>(args);
    end = s.units;
  }
  const int begin = u;

  for (;;) {
    const int j0 = u - s.first, j1 = min(end, s.first + s.units) - s.first;
    int cols;
    {
      const PagedAttnArgs a = fresh_args();
      cols = min(kPaCols, a.cols - s.tile * kPaCols);
      const int n = s.tile * kPaCols + min(kHalf ? c % (kPaCols / 2) : c, cols - 1);   // the last repeats
      const int token = column_token(a, n);
      const int head = s.kvh * a.group + n - token * a.group;
      const Limits limits{s.b, s.keys, s.start + tile_first(a, s.tile), s.start + token};
      Wave<D, kFour, W, kHalf> acc;
      acc.load_ids(limits, j0, w, lane);
      u32x4 q[KK];
      const uint16_t* qr = a.q + s.b * a.qs_b + token * a.qs_t + head * a.qs_h;
      // queries of padding may hold anything: 0, so that they are no reason to run again
      const uint32_t q_keep = token < s.live ? a.q_keep : 0;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        q[kk] = *reinterpret_cast<const u32x4*>(qr + KeyTile<D, kFour>::dim(kk, g));
#pragma unroll
        for (int e = 0; e < 4; ++e) q[kk][e] = (q[kk][e] & q_keep) ^ a.q_flip;
      }
      const HeadPages<D, kFour> pages(a, s.kvh);
      acc.template run<false>(pages, limits, q, a.scale_log2, j0, j1, w, lane, c, g);
      if constexpr (kHalf) acc.add_halves();
      if (g == 0) part_m[w][c] = acc.m == -INFINITY ? -INFINITY : acc.m * a.scale_log2;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (kHalf && g >= 2) break;
        if (c == 0) part_l[w][4 * g + r] = acc.l[r];
#pragma unroll
        for (int i = 0; i < D / 16; i += 4)
          *reinterpret_cast<f32x4*>(&part_o[w][4 * g + r][place_of<D>(c, i)]) =
              f32x4{acc.o[i][r], acc.o[i + 1][r], acc.o[i + 2][r], acc.o[i + 3][r]};
      }
      // an infinite value and a part of P that is 0 make NaN: those again, with P as it is
      if constexpr (!kFour) {
        if (acc.any_nan()) {
          acc.load_ids(limits, j0, w, lane);
          acc.template run<true>(pages, limits, q, a.scale_log2, j0, j1, w, lane, c, g);
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              float& held = part_o[w][4 * g + r][place_of<D>(c, i) + i % 4];
              if (held != held) held = acc.o[i][r];
            }
        }
      }
    }
    const PagedAttnArgs a = fresh_args();
    block_sync();
    const bool whole = j0 == 0 && j1 == s.units;
    const int slot = 2 * blockIdx.x + (u == begin ? 0 : 1);
    if (a.grid > 0 && j0 == 0 && threadIdx.x == 0) {
      const int parts = whole ? 1 : run.owner(s.first + s.units - 1) - blockIdx.x + 1;
      a.parts[(s.b * a.kv_heads + s.kvh) * a.col_tiles + s.tile] =
          u32x2{(uint32_t)slot, (uint32_t)parts};
    }
    for (int e = threadIdx.x; e < cols * (D / 4); e += 64 * W) {
      const int col = e / (D / 4), d = (e % (D / 4)) * 4;
      float top = part_m[0][col];
#pragma unroll
      for (int x = 1; x < W; ++x) top = fmaxf(top, part_m[x][col]);
      float sum = 0.0f;
      f32x4 v{};
#pragma unroll
      for (int x = 0; x < W; ++x) {
        const float wt = part_weight(part_m[x][col], top);
        const f32x4 po = *reinterpret_cast<const f32x4*>(&part_o[x][col][d]);
        sum += wt * part_l[x][col];
#pragma unroll
        for (int y = 0; y < 4; ++y) v[y] += wt * po[y];
      }
      const int cn = s.tile * kPaCols + col;
      const int ct = column_token(a, cn);
      if (ct >= s.live) {      // not live: sees nothing, whatever was added
        v = f32x4{};
        sum = 0.0f;
        top = -INFINITY;
      }
      if (whole) {
        const int64_t row = ((int64_t)s.b * a.tokens + ct) * a.q_heads + s.kvh * a.group + cn -
                            ct * a.group;
        const float inv = top == -INFINITY && sum == 0.0f ? 0.0f : 1.0f / sum;
        u32x2 packed;
        packed[0] = pack_bf16x2(v[0] * inv, v[1] * inv);
        packed[1] = pack_bf16x2(v[2] * inv, v[3] * inv);
        *reinterpret_cast<u32x2*>(a.out + row * D + dim_at<D>(d)) = packed;
        if (d == 0 && a.lse) a.lse[row] = (top + __builtin_amdgcn_logf(sum)) * kLn2;
      } else {
        *reinterpret_cast<f32x4*>(a.part_o + ((int64_t)slot * kPaCols + col) * D + d) = v;
        if (d == 0) {
          a.part_ml[(slot * kPaCols + col) * 2] = top;
          a.part_ml[(slot * kPaCols + col) * 2 + 1] = sum;
        }
      }
    }
    u = s.first + j1;
    if (u >= end || !s.next<Shape::kUnit>(a)) return;
    block_sync();                        // the partials are read before they are overwritten
  }
}

// Join of the partial results of the rows. Rows of one workgroup are written already, rows of
// streams without keys are written here. Grid: (workgroups over the query heads, token, sequence).
constexpr int kPaMergeThreads = 256;

struct MergeRow {
  int64_t row;                           // of out and lse
  int col, slot0, parts;
  bool empty;

  __device__ __forceinline__ MergeRow(const PagedAttnArgs& a, int b, int i, int h) {
    row = ((int64_t)b * a.tokens + i) * a.q_heads + h;
    const int kvh = divide(h, a.group, a.inv_group);
    const int n = i * a.group + h - kvh * a.group, tile = n / kPaCols;
    col = n % kPaCols;
    const int start = a.map.starts[b];
    const int count = a.map.counts ? a.map.counts[b] : a.tokens;
    const u32x2 held = a.parts[((int64_t)b * a.kv_heads + kvh) * a.col_tiles + tile];
    empty = tile_keys(a, start, live_tokens(a, start, count), tile) == 0;
    slot0 = (int)min(held[0], 2u * a.grid - 1);                 // in bounds whatever it holds
    parts = min((int)held[1], a.grid - slot0 / 2);
  }
  // The stream is the first one of every workgroup but perhaps the first.
  __device__ __forceinline__ int slot(int x) const {
    return (x == 0 ? slot0 : (slot0 & ~1) + 2 * x) * kPaCols + col;
  }
};

// Many rows: one wave each, lanes over the dims (and pairs of partials at D = 128).
template <int D>
__global__ __launch_bounds__(kPaMergeThreads) void paged_merge_rows_kernel(PagedAttnArgs a) {
  constexpr int kLanes = D / 4, kGroups = kWave / kLanes;
  constexpr int kAtOnce = 4;             // partials of a lane in flight
  const int lane = threadIdx.x & 63, h = blockIdx.x * (kPaMergeThreads / kWave) + threadIdx.x / kWave;
  if (h >= a.q_heads) return;
  const int dim = lane % kLanes * 4, gr = lane / kLanes;
  for (int b = blockIdx.z; b < a.batch; b += gridDim.z) {
    for (int i = blockIdx.y; i < a.tokens; i += gridDim.y) {
      const MergeRow r(a, b, i, h);
      if (r.empty) {
        if (gr == 0) *reinterpret_cast<u32x2*>(a.out + r.row * D + dim) = u32x2{};
        if (lane == 0 && a.lse) a.lse[r.row] = -INFINITY;
        continue;
      }
      if (r.parts <= 1) continue;
      float top = -INFINITY, sum = 0.0f;
      f32x4 acc{};
      for (int x0 = 0; x0 < r.parts; x0 += kWave) {              // 64 partials at a time
        const int count = min(kWave, r.parts - x0);
        float m = -INFINITY, l = 0.0f;
        if (lane < count) {
          const float* ml = a.part_ml + (int64_t)r.slot(x0 + lane) * 2;
          m = ml[0];
          l = ml[1];
        }
        float higher = fmaxf(top, m);
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) higher = fmaxf(higher, __shfl_xor(higher, o));
        const float old = part_weight(top, higher), wt = part_weight(m, higher);
        sum = sum * old + wave_sum(wt * l);
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[y] *= old;
        top = higher;
        for (int x = 0; x < count; x += kGroups * kAtOnce) {
          f32x4 po[kAtOnce];
#pragma unroll
          for (int k = 0; k < kAtOnce; ++k) {
            const int at = min(x + kGroups * k + gr, count - 1);
            po[k] = *reinterpret_cast<const f32x4*>(a.part_o + (int64_t)r.slot(x0 + at) * D + dim);
          }
#pragma unroll
          for (int k = 0; k < kAtOnce; ++k) {
            const int at = x + kGroups * k + gr;
            const float w = __shfl(wt, min(at, count - 1));
#pragma unroll
            for (int y = 0; y < 4; ++y) acc[y] += at < count ? w * po[k][y] : 0.0f;
          }
        }
      }
      if constexpr (kGroups == 2)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[y] += xor32(acc[y]);
      const float inv = top == -INFINITY && sum == 0.0f ? 0.0f : 1.0f / sum;
      if (gr == 0)
        *reinterpret_cast<u32x2*>(a.out + r.row * D + dim_at<D>(dim)) =
            u32x2{pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv)};
      if (lane == 0 && a.lse) a.lse[r.row] = (top + __builtin_amdgcn_logf(sum)) * kLn2;
    }
  }
}

// Few rows of many partials: one workgroup per (row, 64 dims), the partials in turn over 16 groups
// of threads.
constexpr int kPaMergeDims = 64;

template <int D>
__global__ __launch_bounds__(kPaMergeThreads) void paged_merge_kernel(PagedAttnArgs a) {
  constexpr int kLanes = kPaMergeDims / 4, kGroups = kPaMergeThreads / kLanes, kEarly = 4;
  __shared__ float weight[kPaMaxGrid];
  __shared__ float red[2][kPaMergeThreads / 64];
  __shared__ __align__(16) float acc_s[kGroups][kPaMergeDims];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int d0 = blockIdx.x % (D / kPaMergeDims) * kPaMergeDims;
  const MergeRow r(a, blockIdx.z, blockIdx.y, blockIdx.x / (D / kPaMergeDims));
  const int dim = d0 + tid % kLanes * 4, gr = tid / kLanes;
  if (r.empty) {
    if (gr == 0) *reinterpret_cast<u32x2*>(a.out + r.row * D + dim) = u32x2{};
    if (tid == 0 && d0 == 0 && a.lse) a.lse[r.row] = -INFINITY;
    return;
  }
  if (r.parts <= 1) return;
  // a thread's first partials are under way while the weights are formed
  f32x4 early[kEarly];
#pragma unroll
  for (int k = 0; k < kEarly; ++k) {
    const int x = min(gr + kGroups * k, r.parts - 1);
    early[k] = *reinterpret_cast<const f32x4*>(a.part_o + (int64_t)r.slot(x) * D + dim);
  }
  float top = -INFINITY;
  for (int x = tid; x < r.parts; x += kPaMergeThreads)
    top = fmaxf(top, a.part_ml[(int64_t)r.slot(x) * 2]);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (lane == 0) red[0][w] = top;
  block_sync();
  top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  float sum = 0.0f;
  for (int x = tid; x < r.parts; x += kPaMergeThreads) {
    const float* ml = a.part_ml + (int64_t)r.slot(x) * 2;
    const float wt = part_weight(ml[0], top);
    weight[x] = wt;
    sum += wt * ml[1];
  }
  sum = wave_sum(sum);
  if (lane == 0) red[1][w] = sum;
  block_sync();
  f32x4 acc{};
#pragma unroll
  for (int k = 0; k < kEarly; ++k) {
    const int x = gr + kGroups * k;
    if (x < r.parts)
#pragma unroll
      for (int y = 0; y < 4; ++y) acc[y] += weight[x] * early[k][y];
  }
#pragma unroll 4
  for (int x = gr + kGroups * kEarly; x < r.parts; x += kGroups) {
    const f32x4 po = *reinterpret_cast<const f32x4*>(a.part_o + (int64_t)r.slot(x) * D + dim);
#pragma unroll
    for (int y = 0; y < 4; ++y) acc[y] += weight[x] * po[y];
  }
  *reinterpret_cast<f32x4*>(&acc_s[gr][dim - d0]) = acc;
  block_sync();
  sum = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  if (tid < kPaMergeDims / 2) {
    const float inv = top == -INFINITY && sum == 0.0f ? 0.0f : 1.0f / sum;
    float x = 0.0f, y = 0.0f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      x += acc_s[g][2 * tid];
      y += acc_s[g][2 * tid + 1];
    }
    const int place = d0 + 2 * tid;
    *reinterpret_cast<uint32_t*>(a.out + r.row * D + dim_at<D>(place) + place % 4) =
        pack_bf16x2(x * inv, y * inv);
  }
  if (tid == 0 && d0 == 0 && a.lse) a.lse[r.row] = (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

// ------------------------------------------------------------------------------- host

// Rows from which on a wave joins each: 2048 rows of 2 or 3 partials 78 -> 73 us for both
// kernels, 1024 equal; 64 rows of 128 partials 21 against 41 us.
constexpr int kPaWaveRows = 1024;

// Workgroups (of four waves) that share the units, or 0: one of eight waves per stream and no
// second launch. At 28/4 heads in bf16, 500 keys: 9.7 us so, 9.4 shared, but 2 us less on the host;
// 1090 keys: 14.7 and 9.1 (a step of the eight waves is about 2 us). A launch has fewer than 2^32
// threads: more streams than that share their units, however short.
template <int D, bool kFour>
static int paged_grid(int64_t keys, int64_t streams) {
  if (keys <= 2 * PagedShape<D, kFour, 8>::kUnit && streams <= 0xffffffffll / 512) return 0;
  using Shape = PagedShape<D, kFour, 4>;
  const int64_t units = (keys + Shape::kUnit - 1) / Shape::kUnit;
  return (int)std::min<int64_t>(std::min(kPaMaxGrid, kPaCus * Shape::kPerCu), streams * units);
}

struct PagedSizes {
  int64_t keys, streams, rows;
};

static bool paged_sizes(const spx_paged_cache& z, int q_heads, int max_keys, PagedSizes& s) {
  if (z.table_width <= 0 || z.page_size <= 0 || max_keys < 0 || z.batch <= 0 || z.tokens <= 0 ||
      q_heads <= 0 || q_heads > 1 << 20 || z.kv_heads <= 0 || q_heads % z.kv_heads != 0)
    return false;
  if ((double)z.batch * z.tokens * q_heads > 0x7fffffff) return false;
  s.rows = (int64_t)z.batch * z.tokens * q_heads;
  s.keys = (int64_t)z.table_width * z.page_size;
  const int64_t cols = (int64_t)z.tokens * (q_heads / z.kv_heads);
  s.streams = (int64_t)z.batch * z.kv_heads * ((cols + kPaCols - 1) / kPaCols);
  // units are counted in 32 bits, also where max_keys is no bound after all
  if ((s.keys + kPaMinUnit - 1) / kPaMinUnit > 0x7fffffff / s.streams) return false;
  if (max_keys > 0) s.keys = std::min<int64_t>(s.keys, max_keys);
  return true;
}

static int paged_grid_of(const PagedSizes& z, int head_dim, bool four) {
  if (head_dim == 128)
    return four ? paged_grid<128, true>(z.keys, z.streams) : paged_grid<128, false>(z.keys, z.streams);
  return four ? paged_grid<256, true>(z.keys, z.streams) : paged_grid<256, false>(z.keys, z.streams);
}

template <int D, bool kFour>
static int launch_paged(PagedAttnArgs a, const PagedSizes& z, void* workspace, hipStream_t st) {
  if (a.grid == 0) {
    const unsigned streams = (unsigned)z.streams;
    paged_attn_kernel<D, kFour, 8, false><<<streams, 512, 0, st>>>(a);
    return launch_status("paged_attention");
  }
  SPX_REQUIRE(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, SPX_EINVAL,
              "paged_attention: workspace null or not 16-byte aligned");
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + (int64_t)2 * a.grid * kPaCols * D;
  a.parts = reinterpret_cast<u32x2*>(a.part_ml + (int64_t)2 * a.grid * kPaCols * 2);
  const unsigned grid = (unsigned)a.grid;
  // The half form where workgroups may run long: 64 sequences of 8192 keys (32/8 heads) 123 -> 121
  // us; with two parts of P a workgroup's one unit of 32641 keys (28/4) took 12.4 instead of 11.8 in
  // it, and D = 256 was as fast without it (44.1 and 44.3 us).
  constexpr bool kCanHalve = D == 128 && kFour;
  const int64_t units = z.streams * ((z.keys + PagedShape<D, kFour, 4>::kUnit - 1) /
                                     PagedShape<D, kFour, 4>::kUnit);
  if (kCanHalve && a.cols <= kPaCols / 2 && units >= (int64_t)8 * a.grid)
    paged_attn_kernel<D, kFour, 4, kCanHalve><<<grid, 256, 0, st>>>(a);
  else paged_attn_kernel<D, kFour, 4, false><<<grid, 256, 0, st>>>(a);
  if (z.rows >= kPaWaveRows || a.batch > 65535 || a.tokens > 65535) {
    const int waves = kPaMergeThreads / kWave;
    paged_merge_rows_kernel<D><<<dim3((unsigned)((a.q_heads + waves - 1) / waves),
                                      (unsigned)std::min(a.tokens, 65535),
                                      (unsigned)std::min(a.batch, 65535)),
                                 kPaMergeThreads, 0, st>>>(a);
  } else {
    paged_merge_kernel<D><<<dim3((unsigned)(a.q_heads * (D / kPaMergeDims)), (unsigned)a.tokens,
                                 (unsigned)a.batch),
                            kPaMergeThreads, 0, st>>>(a);
  }
  return launch_status("paged_attention");
}

}  // namespace spx

using namespace spx;

extern "C" int64_t spx_paged_attention_workspace_bytes(const spx_paged_cache* cache, int q_heads,
                                                       int max_keys) {
  PagedSizes z;
  if (cache == nullptr || !paged_sizes(*cache, q_heads, max_keys, z) ||
      (cache->head_dim != 128 && cache->head_dim != 256))
    return -1;
  const int grid = paged_grid_of(z, cache->head_dim, cache->key_scales != nullptr);
  return grid == 0 ? 0 : (int64_t)2 * grid * kPaCols * (cache->head_dim + 2) * 4 + z.streams * 8;
}

extern "C" int spx_paged_attention(const spx_paged_cache* cache, const void* q,
                                   const int64_t* q_strides, int q_heads, int max_keys, float scale,
                                   void* workspace, void* out, float* lse, void* stream) {
  PagedAttnArgs a{};
  const int status = paged_map(a.map, cache);
  if (status != SPX_OK) return status;
  PagedSizes z;
  SPX_REQUIRE(paged_sizes(*cache, q_heads, max_keys, z), SPX_EINVAL,
              "bad shape: batch %d tokens %d q_heads %d kv_heads %d max_keys %d", cache->batch,
              cache->tokens, q_heads, cache->kv_heads, max_keys);
  SPX_REQUIRE(q && q_strides && out, SPX_EINVAL, "null pointer");
  SPX_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0 &&
                  q_strides[3] == 1 && ((q_strides[0] | q_strides[1] | q_strides[2]) & 7) == 0,
              SPX_EINVAL,
              "q, out: bases must be 16-byte aligned, q's dim stride 1, the others multiples of 8");
  const bool four = cache->key_scales != nullptr;
  a.q = static_cast<const uint16_t*>(q);
  a.qs_b = q_strides[0]; a.qs_t = q_strides[1]; a.qs_h = q_strides[2];
  a.key_pages = cache->key_pages; a.value_pages = cache->value_pages;
  a.key_scales = static_cast<const uint8_t*>(cache->key_scales);
  a.value_scales = static_cast<const uint8_t*>(cache->value_scales);
  a.batch = cache->batch; a.tokens = cache->tokens;
  a.q_heads = q_heads; a.kv_heads = cache->kv_heads; a.group = q_heads / cache->kv_heads;
  a.cols = cache->tokens * a.group;
  a.col_tiles = (a.cols + kPaCols - 1) / kPaCols;
  a.grid = paged_grid_of(z, cache->head_dim, four);
  a.inv_grid = 1.0 / std::max(a.grid, 1);
  a.inv_group = 1.0 / a.group;
  a.scale_log2 = scale == 0 ? 1.0f : (float)(std::abs((double)scale) * 1.4426950408889634);
  a.q_keep = scale == 0 ? 0 : 0xffffffffu;
  a.q_flip = scale < 0 ? 0x80008000u : 0;
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (cache->head_dim == 128)
    return four ? launch_paged<128, true>(a, z, workspace, st)
                : launch_paged<128, false>(a, z, workspace, st);
  return four ? launch_paged<256, true>(a, z, workspace, st)
              : launch_paged<256, false>(a, z, workspace, st);
}
