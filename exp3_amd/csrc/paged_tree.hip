// Attention of a tree of drafted tokens over a paged KV cache (bf16 or 4-bit pages; bf16 queries
// and outputs, fp32 scores, softmax and accumulation), and the tree's plan.
//
// New token i of a sequence (in place starts + i) sees the places below `starts` and the new tokens j
// of bit j of its mask: with m and l the running maximum and sum of its scores x = scale q k,
//   O <- O e^(m - m') + sum e^(x - m') v,   l <- l e^(m - m') + sum e^(x - m'),   out = O / l.
//
// Columns n = i group + h of a KV head (token i of T, query head h of the group) share its K and V;
// 64 or 128 of them are one tile. A stream is a (sequence, KV head, column tile), its work
// ceil(keys / 64) units of 64 keys, and the units of all streams are dealt in equal runs to one grid
// (lengths are device data); a second kernel joins the partial results of the streams that
// workgroups share.
//
// Between HBM and the matrix units: at 128 columns a unit's products take half as long as its bytes in
// bf16, twice as long in 4 bits. So K and V are read once for 128 columns and are on their way a unit
// and a half ahead, and a wave's softmax, or its widening of 4 bits, is issued between products. P goes
// to the products in two bf16 parts, which lose up to 2^-17 of it: an output is off by up to 2^-17 of
// the sum of p |v|, and 0.12 % of the outputs round otherwise than the plain fp32 form's. With a third
// part it is 0.03 to 0.08 %, the order of the sums, for 5 to 17 % more time (in a graph 87.9 -> 103, 4
// bits 113 -> 132, D = 256 50.2 -> 54.0 us). One part would save a third of the matrix instructions and
// lose up to 2^-8, as much as the output's own rounding.
//
// 8 ragged sequences of up to 16000 keys, trees of 32, 32/8 heads, bf16: 79 us (4.0 TB/s) + 11 to join;
// 16 of up to 8192 in 4 bits, trees of 61, 28/4 heads: 101 (0.47 PFLOP/s, 0.71 with both parts of P) + 11;
// 4 of up to 12001 at D = 256, trees of 26, 16/4 heads: 40 + 9 in 4 bits and in bf16, one wave per SIMD
// (LDS). The plan of a tree (below): 16 nodes 1.8 us, 64 trees of 61 3.2.
#include <algorithm>
#include <cmath>

#include "paged_tiles.h"

namespace spx {

constexpr int kTreeMaxTokens = 256;
constexpr int kTreeKeys = 64;            // keys of a unit
constexpr int kTreeThreads = 256;
constexpr int kTreeCus = 256;

typedef short s16x4 __attribute__((ext_vector_type(4)));

template <int D>
struct TreeShape {
  static constexpr int kPerCu = D == 128 ? 2 : 1;              // resident workgroups (LDS)
  static constexpr int kRow = 2 * D;                           // bytes of a row in LDS
  static constexpr int kTile = kTreeKeys * kRow;
};

struct TreeArgs {
  PagedMap map;
  const uint16_t* q;
  int64_t qs_b, qs_t, qs_h;
  const void* key_pages;
  const void* value_pages;
  const uint8_t* key_scales;
  const uint8_t* value_scales;
  const uint64_t* masks;                 // [B, T, words]
  int words;
  int batch, tokens, q_heads, kv_heads, group;
  int cols, col_tiles;                   // tokens x group, tiles of them
  int grid;                              // workgroups sharing the units
  double inv_grid, inv_group;            // reciprocals
  float scale_log2;                      // > 0: the sign of the scale, or a scale of 0, goes to q
  uint32_t q_keep, q_flip;               // q & q_keep ^ q_flip
  uint16_t* out;
  float* lse;
  float* part_o;                         // [2 grid][D / 4][columns of a tile][4]
  float* part_ml;                        // [2 grid][columns of a tile][2]
  u32x2* parts;                          // [streams] first partial's slot, how many (1: written out)
};

// Live tokens of a sequence: 0 .. live - 1.
__device__ __forceinline__ int tree_live(const TreeArgs& a, int start, int count) {
  const int64_t room = a.map.capacity() - start;
  const int live = min(min(count, a.tokens), (int)min(room, (int64_t)a.tokens));
  return start < 0 ? 0 : max(live, 0);
}

// A sequence's streams: `tiles` for each KV head, of `units` units.
struct TreeLengths {
  int start, live, keys, tiles, units;
  __device__ __forceinline__ void of(const TreeArgs& a, int columns, int start_, int count) {
    start = start_;
    live = tree_live(a, start, count);
    keys = live > 0 ? start + live : 0;
    tiles = (live * a.group + columns - 1) / columns;
    units = (keys + kTreeKeys - 1) / kTreeKeys;
  }
  __device__ __forceinline__ void load(const TreeArgs& a, int columns, int b) {
    of(a, columns, scalar_load(a.map.starts + b),
       a.map.counts ? scalar_load(a.map.counts + b) : a.tokens);
  }
};

struct TreeScan {                        // the units of 64 sequences, one a lane
  int units, sum;
  __device__ __forceinline__ void load(const TreeArgs& a, int columns, int b) {
    TreeLengths x;
    int start = -1, count = a.tokens;
    if (b < a.batch) {
      start = a.map.starts[b];
      if (a.map.counts) count = a.map.counts[b];
    }
    x.of(a, columns, start, count);
    units = x.tiles * x.units * a.kv_heads;
    sum = wave_prefix(units);
  }
  __device__ __forceinline__ int total() const { return __builtin_amdgcn_readlane(sum, kWave - 1); }
};

struct TreeStream {
  TreeLengths x;
  int b, kvh, tile, first;               // first: of its units
  // The stream of unit u; false: there is none (lengths that change under the launch must not make
  // it loop).
  __device__ __forceinline__ bool find(const TreeArgs& a, int columns, int lane, TreeScan scan, int u) {
    int before = 0, b0 = 0;
    uint64_t past;
    while (!(past = __ballot(before + scan.sum > u))) {
      before += scan.total();
      b0 += kWave;
      if (b0 >= a.batch) return false;
      scan.load(a, columns, b0 + lane);
    }
    const int l = __builtin_ctzll(past);
    b = b0 + l;
    before += __builtin_amdgcn_readlane(scan.sum - scan.units, l);
    x.load(a, columns, b);
    if (x.units <= 0 || u < before) return false;
    const int at = (u - before) / x.units;
    kvh = at / x.tiles;
    tile = at - kvh * x.tiles;
    first = before + at * x.units;
    return kvh < a.kv_heads;
  }
  // The next one that has units.
  __device__ __forceinline__ bool next(const TreeArgs& a, int columns) {
    first += x.units;
    if (++tile < x.tiles) return true;
    tile = 0;
    if (++kvh < a.kv_heads) return true;
    kvh = 0;
    do {
      if (++b >= a.batch) return false;
      x.load(a, columns, b);
    } while (x.units == 0);
    return true;
  }
};

struct TreeRun {                         // units begin(w) .. begin(w + 1) - 1 of workgroup w
  int per, rest;
  __device__ __forceinline__ TreeRun(int total, int grid, double inv)
      : per(first_lane(divide(total, grid, inv))), rest(total - per * grid) {}
  __device__ __forceinline__ int begin(int w) const { return w * per + min(w, rest); }
  __device__ __forceinline__ int owner(int u) const {
    const int wide = rest * (per + 1);
    return u < wide ? u / (per + 1) : rest + (u - wide) / max(per, 1);
  }
};

__device__ __forceinline__ uint64_t bits_below(int n) {
  return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1;
}

// Which of the keys key0 .. key0 + 31 a token sees, as bits.
__device__ __forceinline__ uint32_t tree_visible(const TreeArgs& a, int b, int token,
                                                 const TreeLengths& x, int key0) {
  if (token >= x.live) return 0;
  const int o = key0 - x.start;          // of the first one among the new tokens
  if (o <= -32) return ~0u;
  const uint64_t* m = a.masks + ((int64_t)b * a.tokens + token) * a.words;
  const int w = max(o, 0) >> 6;
  const uint64_t low = w < a.words ? m[w] & bits_below(x.live - 64 * w) : 0;
  const uint64_t high = w + 1 < a.words ? m[w + 1] & bits_below(x.live - 64 * w - 64) : 0;
  if (o < 0) return (uint32_t)(low << -o) | ((1u << -o) - 1);
  const int s = o & 63;
  return (uint32_t)(low >> s | (s ? high << (64 - s) : 0));
}

// ------------------------------------------------------------------ tiles in LDS
//
// Rows of D bf16 values, 16-byte chunks exchanged within a row by an XOR with tree_swizzle(row). Free
// of bank conflicts are: score operands (one chunk of 16 rows: 16 different chunks), transposing reads
// (four chunks of four rows 4 t .. 4 t + 3: all four 64-byte groups) and the rows widened from 4 bits
// (every fourth chunk of such rows: all 16).
__device__ __forceinline__ int tree_swizzle(int row) {
  return (row & 3) << 2 | ((row ^ row >> 2) & 3);
}

// Four times 16 bytes a lane from base + offset[i] to to + 1024 i + 16 lane, past the registers. From
// assembly: the compiler would wait for its own form of it before any other read of LDS.
__device__ __forceinline__ void copy_to_lds(GlobalBytes base, const uint32_t* offset, LdsBytes to) {
#if defined(__HIP_DEVICE_COMPILE__)
  const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)to);
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %2, %6\n\t"
      "s_add_u32 m0, m0, 0x400\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %3, %6\n\t"
      "s_add_u32 m0, m0, 0x400\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %4, %6\n\t"
      "s_add_u32 m0, m0, 0x400\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %5, %6\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "s"(m0), "v"(offset[0]), "v"(offset[1]), "v"(offset[2]), "v"(offset[3]), "s"(base)
      : "memory", "scc");
#endif
}

// 16 rows of K or V on their way into LDS.
template <int D, bool kFour>
struct TreeRows;

template <int D>
struct TreeRows<D, false> {
  static constexpr int kRow = 2 * D, kLanes = D / 8, kRows = kWave / kLanes;   // rows a copy
  static constexpr int kCopies = 16 / kRows;
  uint32_t offset[kCopies];              // of the lane's 16 bytes from the first row on
  __device__ __forceinline__ TreeRows(int lane) {
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int r = kRows * i + lane / kLanes;
      offset[i] = r * kRow + ((lane % kLanes) ^ tree_swizzle(r)) * 16;
    }
  }
  __device__ __forceinline__ void copy(GlobalBytes pages, int64_t row, LdsBytes to) const {
    const GlobalBytes from = tile_base(pages + row * kRow);
#pragma unroll
    for (int i = 0; i < kCopies; i += 4) copy_to_lds(from, offset + i, to + 1024 * i);
  }
  // Rows from `limit` on become 0.
  static __device__ __forceinline__ void clear(LdsBytes to, int limit, int lane) {
#pragma unroll
    for (int i = 0; i < kCopies; ++i)
      if (kRows * i + lane / kLanes >= limit) lds_store(to, 1024 * i + 16 * lane, u32x4{});
  }
};

template <int D>
struct TreeRows<D, true> {
  static constexpr int kRow = 2 * D, kPieces = D / 32, kRows = kWave / kPieces, kLoads = 16 / kRows;
  u32x4 raw[kLoads];                     // 32 dims of a row: one scale
  uint32_t scale[kLoads];
  __device__ __forceinline__ void load(GlobalBytes pages, GlobalBytes scales, int64_t row, int lane) {
    const GlobalBytes p = tile_base(pages + row * (D / 2)),
                      s = tile_base(scales + row * (D / kPagedGroup));
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      raw[i] = global_load<u32x4>(p, 1024 * i + 16 * lane);
      scale[i] = global_load<uint8_t>(s, 64 * i + lane);
    }
  }
  // Rows from `limit` on become 0.
  __device__ __forceinline__ void limit(int rows, int lane) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      if (kRows * i + lane / kPieces >= rows) {
        raw[i] = u32x4{};
        scale[i] = 127;
      }
  }
  static constexpr int kParts = 4 * kLoads;
  // Part n of them (8 dims a lane) widened into LDS.
  __device__ __forceinline__ void store(LdsBytes to, int n, int lane) const {
    const int i = n / 4, y = n % 4, r = kRows * i + lane / kPieces, piece = lane % kPieces;
    lds_store(to, r * kRow + ((4 * piece + y) ^ tree_swizzle(r)) * 16,
              widen8(raw[i][y], __uint_as_float(scale[i] << 23)));
  }
};

// ------------------------------------------------------------------- main kernel

// A wave's 32 columns: column n in the lanes n and n + 32.
template <int D>
struct TreeState {
  f32x16 o[D / 32];                      // O^T: dim 32 i + mfma32_row(r, lane)
  float m, l;                            // maximum, unscaled; sum over the lane's keys
};

__device__ __forceinline__ float other_half_max(float x) {
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
}
__device__ __forceinline__ float other_half_sum(float x) {
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

// Nothing is scheduled across it: operands are read a few products ahead and stay so.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// K rows as A operands: lane n holds row n % 32.
template <int D>
struct TreeKeys {
  LdsBytes row;
  int at;
  __device__ __forceinline__ TreeKeys(LdsBytes k, int lane)
      : row(k + (lane & 31) * (2 * D)), at(((lane >> 5) ^ tree_swizzle(lane & 31)) << 4) {}
  __device__ __forceinline__ u32x4 operand(int kk) const {
    return lds_load<u32x4>(row, at ^ (kk << 5));
  }
};

// V^T of 32 dims and 16 keys as A operands, read transposed: lane 16 g + 4 e + a reads four dims of
// key e of its group's four, lane L of a group receives dim L of all four.
template <int D>
struct TreeValues {
  LdsBytes base;
  int at;
  __device__ __forceinline__ TreeValues(LdsBytes v, int lane) {
    const int e = lane >> 2 & 3, a = lane & 3, g = lane >> 4;
    const int row = 4 * (lane >> 5) + e;
    base = v + row * (2 * D) + 8 * (a & 1);
    at = ((2 * (g & 1) + (a >> 1)) ^ tree_swizzle(row)) << 4;
  }
  // t: block t % (D / 32) of the dims, keys 16 (t / (D / 32)) ..
  __device__ __forceinline__ u32x4 operand(int t) const {
    const int kc = t / (D / 32), i = t % (D / 32);
    u32x4 vt;
#pragma unroll
    for (int s = 0; s < 2; ++s) {        // rows 8 further on: bit 1 of the swizzle
      const u32x2 part = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                     (__attribute__((address_space(3))) s16x4*)(
                         base + (16 * kc + 8 * s) * (2 * D) + (at ^ (64 * i) ^ (32 * s)))));
      vt[2 * s] = part[0];
      vt[2 * s + 1] = part[1];
    }
    return vt;
  }
};

// O by corr, in place and from assembly: the compiler makes the products of a branch, and as many
// selections, part of every step. It does not see that matrix instructions wrote O: 19 wait states
// before it is read.
template <int D>
__device__ __forceinline__ void tree_rescale(TreeState<D>& st, float corr) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 2");
#pragma unroll
  for (auto& o : st.o)
#pragma unroll
    for (int r = 0; r < 16; ++r) asm volatile("v_mul_f32 %0, %0, %1" : "+v"(o[r]) : "v"(corr));
#endif
}

// P of 32 keys in two bf16 parts, operands of two products over 16 keys each. Of a P in [2^e, 2^(e + 1))
// the first part leaves up to 2^(e - 8), half a step, and the second, whose half steps are 2^-9 of that
// or finer, up to 2^(e - 17). The sums take P as it is.
struct TreeProbs {
  u32x4 hi[2], lo[2];
};

// Scores that a column does not see become -inf.
__device__ __forceinline__ void tree_mask(f32x16& x, uint32_t seen, int lane) {
  const uint32_t mine = seen >> (4 * (lane >> 5));
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (!(mine >> (8 * (r / 4) + r % 4) & 1)) x[r] = -INFINITY;
}

// The running maximum takes in x: what O and l are to be multiplied by, or 1.
template <int D>
__device__ __forceinline__ bool tree_raise(TreeState<D>& st, const f32x16& x, float scale, float& corr) {
  float mx = x[0];
#pragma unroll
  for (int r = 1; r < 16; ++r) mx = fmaxf(mx, x[r]);
  mx = other_half_max(mx);
  corr = 1.0f;
  if (!__any(mx > st.m)) return false;
  const float m_new = fmaxf(st.m, mx);
  corr = st.m == -INFINITY ? 0.0f : exp2_fast((st.m - m_new) * scale);
  st.m = m_new;
  st.l *= corr;
  return true;
}

struct TreeNothing {
  __device__ __forceinline__ void operator()(int = 0) const {}
};

// P from the scores x of 32 keys; beside it, kScores: the scores `next` of other keys, kProducts: the
// products of V with the P of other keys. A wave issues a vector instruction every five cycles or so
// while a product takes 32, so each is followed by its share of the others' work.
template <int D, bool kScores, bool kProducts>
__device__ __forceinline__ void tree_softmax(TreeState<D>& st, const u32x4 (&q)[D / 16],
                                             const TreeKeys<D>& keys, const TreeValues<D>& values,
                                             float scale, f32x16& x, f32x16& next, TreeProbs& p,
                                             const TreeProbs& last) {
  constexpr int kSteps = D / 16, kAhead = 2;
  u32x4 key_ring[kAhead], value_ring[kAhead];
#pragma unroll
  for (int t = 0; t < kAhead; ++t) {
    if constexpr (kScores) key_ring[t] = keys.operand(t);
    if constexpr (kProducts) value_ring[t] = values.operand(t);
  }
  if constexpr (kScores) next = f32x16{};
  const float shift = st.m == -INFINITY ? 0.0f : st.m * scale;
  // sums of two: their error grows with the number of steps alone
  float sum[8];
  fence();
#pragma unroll
  for (int t = 0; t < kSteps; ++t) {
    const int kc = t / (D / 32), i = t % (D / 32);
    const int pair = t * 8 / kSteps, r = 2 * pair;             // of scores, and its first
    const bool first = t * 8 % kSteps == 0, second = (t + 1) * 8 % kSteps == 0;
    u32x4 kt, vt;
    if constexpr (kScores) kt = key_ring[t % kAhead];
    if constexpr (kProducts) {
      vt = value_ring[t % kAhead];
      st.o[i] = mfma32(as_bf16x8(vt), as_bf16x8(last.hi[kc]), st.o[i]);
    }
    if (first) {
      x[r] = exp2_fast(__builtin_fmaf(x[r], scale, -shift));
      x[r + 1] = exp2_fast(__builtin_fmaf(x[r + 1], scale, -shift));
    }
    if constexpr (kScores)
      if (t + kAhead < kSteps) key_ring[t % kAhead] = keys.operand(t + kAhead);
    if constexpr (kProducts) fence();
    if constexpr (kScores) next = mfma32(as_bf16x8(kt), as_bf16x8(q[t]), next);
    if (second) {
      const uint32_t w = (uint32_t)opaque((int)pack_bf16x2(x[r], x[r + 1]));
      p.hi[r / 8][r / 2 % 4] = w;
      sum[pair] = x[r] + x[r + 1];
      x[r] -= bf16_lo(w);
      x[r + 1] -= bf16_hi(w);
    }
    if constexpr (kProducts) {
      fence();
      st.o[i] = mfma32(as_bf16x8(vt), as_bf16x8(last.lo[kc]), st.o[i]);
    }
    // (opaque: else it is made where it is used)
    if (second) p.lo[r / 8][r / 2 % 4] = (uint32_t)opaque((int)pack_bf16x2(x[r], x[r + 1]));
    if constexpr (kProducts)
      if (t + kAhead < kSteps) value_ring[t % kAhead] = values.operand(t + kAhead);
    fence();
  }
#pragma unroll
  for (int n = 4; n >= 1; n /= 2)
#pragma unroll
    for (int r = 0; r < n; ++r) sum[r] += sum[r + n];
  st.l += sum[0];
}

// Products with V alone; extra(t): other work beside product t of D / 16.
template <int D, typename Extra>
__device__ __forceinline__ void tree_products(TreeState<D>& st, const TreeValues<D>& values,
                                              const TreeProbs& p, const Extra& extra) {
  constexpr int kSteps = D / 16, kAhead = 2;
  u32x4 ring[kAhead];
#pragma unroll
  for (int t = 0; t < kAhead; ++t) ring[t] = values.operand(t);
  fence();
#pragma unroll
  for (int t = 0; t < kSteps; ++t) {
    const int kc = t / (D / 32), i = t % (D / 32);
    const u32x4 vt = ring[t % kAhead];
    st.o[i] = mfma32(as_bf16x8(vt), as_bf16x8(p.hi[kc]), st.o[i]);
    st.o[i] = mfma32(as_bf16x8(vt), as_bf16x8(p.lo[kc]), st.o[i]);
    if (t + kAhead < kSteps) ring[t % kAhead] = values.operand(t + kAhead);
    extra(t);
    fence();
  }
}

template <int D>
__device__ __forceinline__ f32x16 tree_scores(const u32x4 (&q)[D / 16], const TreeKeys<D>& keys) {
  constexpr int kSteps = D / 16, kAhead = 4;
  u32x4 ring[kAhead];
#pragma unroll
  for (int t = 0; t < kAhead; ++t) ring[t] = keys.operand(t);
  f32x16 x{};
  fence();
#pragma unroll
  for (int t = 0; t < kSteps; ++t) {
    x = mfma32(as_bf16x8(ring[t % kAhead]), as_bf16x8(q[t]), x);
    if (t + kAhead < kSteps) ring[t % kAhead] = keys.operand(t + kAhead);
    fence();
  }
  return x;
}

// NS blocks of 32 keys of a unit. With two, the scores of the second are formed beside the first's
// softmax, and the first's products beside the second's. middle(): K has been read, V is read next.
template <int D, int NS, typename Middle, typename Extra>
__device__ __forceinline__ void tree_unit(TreeState<D>& st, const u32x4 (&q)[D / 16], LdsBytes k,
                                          LdsBytes v, float scale, bool masked,
                                          const uint32_t (&seen)[NS], int lane, const Middle& middle,
                                          const Extra& extra) {
  constexpr int kBlock = 32 * 2 * D;
  float corr;
  const TreeValues<D> values(v, lane);
  f32x16 x = tree_scores<D>(q, TreeKeys<D>(k, lane));
  if (masked) tree_mask(x, seen[0], lane);
  if (tree_raise<D>(st, x, scale, corr)) tree_rescale<D>(st, corr);
  TreeProbs p;
  if constexpr (NS == 1) {
    f32x16 none;
    tree_softmax<D, false, false>(st, q, TreeKeys<D>(k, lane), values, scale, x, none, p, p);
    middle();
    tree_products<D>(st, values, p, extra);
  } else {
    f32x16 y, none;
    tree_softmax<D, true, false>(st, q, TreeKeys<D>(k + kBlock, lane), values, scale, x, y, p, p);
    middle();
    if (masked) tree_mask(y, seen[1], lane);
    const bool grows = tree_raise<D>(st, y, scale, corr);
    TreeProbs p1;
    tree_softmax<D, false, true>(st, q, TreeKeys<D>(k, lane), values, scale, y, none, p1, p);
    if (grows) tree_rescale<D>(st, corr);
    tree_products<D>(st, TreeValues<D>(v + kBlock, lane), p1, extra);
  }
}

// Block by block, each product with V by itself in fp32 and only into columns that see the key: an
// infinite or NaN value does not reach others, and meets no part of a P that is 0.
template <int D, int NS>
__device__ __forceinline__ void tree_careful_unit(TreeState<D>& st, const u32x4 (&q)[D / 16], LdsBytes k,
                                                  LdsBytes v, float scale, const uint32_t (&seen)[NS],
                                                  int lane) {
#pragma unroll 1
  for (int s = 0; s < NS; ++s) {
    const uint32_t sees = NS == 2 && s == 1 ? seen[NS - 1] : seen[0];
    f32x16 x = tree_scores<D>(q, TreeKeys<D>(k + s * 64 * D, lane));
    tree_mask(x, sees, lane);
    float corr;
    if (tree_raise<D>(st, x, scale, corr)) tree_rescale<D>(st, corr);
    const float shift = st.m == -INFINITY ? 0.0f : st.m * scale;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] = exp2_fast(__builtin_fmaf(x[r], scale, -shift));
      st.l += x[r];
    }
#pragma unroll 1
    for (int key = 0; key < 32; ++key) {
      float mine = 0.0f;                 // P of the key, where this lane has it
#pragma unroll
      for (int r = 0; r < 16; ++r) mine = mfma32_row(r, lane) == key ? x[r] : mine;
      const float p = __shfl(mine, (key >> 2 & 1) * 32 + (lane & 31));
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const int d = 32 * i + mfma32_row(r, lane);
          const u32x2 w = lds_load<u32x2>(v, (32 * s + key) * (2 * D) +
                                                 ((d >> 3 ^ tree_swizzle(key)) << 4) + (d & 7) * 2);
          const float value[4] = {bf16_lo(w[0]), bf16_hi(w[0]), bf16_lo(w[1]), bf16_hi(w[1])};
#pragma unroll
          for (int y = 0; y < 4; ++y) st.o[i][r + y] += sees >> key & 1 ? p * value[y] : 0.0f;
        }
    }
  }
}

// Of two workgroups on a CU the older goes first at every issue, ends first and leaves the younger alone.
// So they take turns at the higher priority, 8192 cycles each. (Without and with: 8 ragged sequences
// of up to 16000 tokens, trees of 32, 32/8 heads, 86.3 and 85.8 us; 16 of 8192, 4 bits, trees of 61, 128
// and 124.5 us.)
__device__ __forceinline__ void tree_turn() {
  __builtin_amdgcn_s_setprio(0);
  if ((__builtin_amdgcn_s_memtime() >> 13 ^ blockIdx.x >> 8) & 1) __builtin_amdgcn_s_setprio(2);
}

// Units j .. end - 1 of a stream. WK waves share a column group's keys.
template <int D, bool kFour, int WC, bool kCareful>
__device__ __forceinline__ void tree_run(TreeState<D>& st, const TreeArgs& a, const TreeStream& s,
                                         const u32x4 (&q)[D / 16], int token, bool idle, LdsBytes tiles,
                                         int j, int end, int w, int lane) {
  using Shape = TreeShape<D>;
  constexpr int WK = 4 / WC, NS = 2 / WK, kGroups = kTreeKeys / 16, kRow = Shape::kRow;
  const HeadPages<D, kFour> pages(a, s.kvh);
  const int sub = WK == 2 ? w / WC : 0;  // the wave's first block of 32 keys
#pragma unroll
  for (auto& o : st.o) o = f32x16{};
  st.m = -INFINITY;
  st.l = 0.0f;
  // lane i: page of group i % 4 in unit id_base + i / 4
  int id_base = j;
  const auto fetch_ids = [&](int j) {
    const int64_t p = ((int64_t)j + lane / kGroups) * kTreeKeys + lane % kGroups * 16;
    return a.map.page(s.b, (int)min(p, (int64_t)s.x.keys - 1));
  };
  int ids = fetch_ids(j), next_ids = fetch_ids(j + kWave / kGroups);
  uint64_t lost = __ballot(ids < 0);     // groups without a place
  const auto bad_of = [&](int j) { return (uint32_t)(lost >> ((j - id_base) * kGroups)) & 15u; };
  const auto advance = [&](int j) {
    if (j - id_base < kWave / kGroups) return;
    id_base = j;
    ids = next_ids;
    lost = __ballot(ids < 0);
    next_ids = fetch_ids(j + kWave / kGroups);
  };
  const auto row_of = [&](int j) {
    const int id = max(__builtin_amdgcn_readlane(ids, (j - id_base) * kGroups + w), 0);
    return pages.row(id, j * kTreeKeys + 16 * w);
  };
  // tile 0 / 1 of a buffer: K / V; a wave feeds group w of both
  const auto tile = [&](int buffer, int which) { return tiles + (2 * buffer + which) * Shape::kTile; };
  const auto place = [&](int buffer, int which) { return tile(buffer, which) + 16 * w * kRow; };
  const auto rows_left = [&](int j, uint32_t bad) {
    return bad >> w & 1 ? 0 : s.x.keys - j * kTreeKeys - 16 * w;
  };
  const auto compute = [&](int j, int buffer, uint32_t bad, const auto& middle, const auto& extra) {
    const int first = j * kTreeKeys + 32 * sub;
    const bool masked = bad != 0 || first + 32 * NS > s.x.start;
    uint32_t seen[NS];
#pragma unroll
    for (int y = 0; y < NS; ++y) {
      seen[y] = ~0u;
      if (!masked) continue;
      seen[y] = tree_visible(a, s.b, token, s.x, first + 32 * y);
      if (bad >> (2 * (sub + y)) & 1) seen[y] &= 0xffff0000u;
      if (bad >> (2 * (sub + y) + 1) & 1) seen[y] &= 0xffffu;
    }
    const LdsBytes k = tile(buffer, 0) + 32 * sub * kRow, v = tile(buffer, 1) + 32 * sub * kRow;
    if constexpr (kCareful)
      tree_careful_unit<D, NS>(st, q, k, v, a.scale_log2, seen, lane);
    else
      tree_unit<D, NS>(st, q, k, v, a.scale_log2, masked, seen, lane, middle, extra);
  };
  if constexpr (!kFour && kCareful) {
    const TreeRows<D, false> rows(lane);
    for (; j < end; ++j) {
      advance(j);
      const int64_t row = row_of(j);
      rows.copy(pages.keys, row, place(0, 0));
      rows.copy(pages.values, row, place(0, 1));
      const uint32_t bad = bad_of(j);
      const int left = rows_left(j, bad);
      wait_copies<0>();
      if (left < 16) TreeRows<D, false>::clear(place(0, 1), left, lane);
      block_sync();
      if (!idle) compute(j, 0, bad, TreeNothing(), TreeNothing());
      block_sync();
    }
  } else if constexpr (!kFour) {
    // K of unit j + 2 comes in from the middle of unit j on, where K of unit j has been read, V of unit
    // j + 1 from the beginning of unit j on: each for one and a half units, 48 KB a workgroup at D =
    // 128.
    constexpr int kCopies = TreeRows<D, false>::kCopies;
    const TreeRows<D, false> rows(lane);
    int64_t next_row = row_of(j);        // of the unit whose K went last
    uint32_t bad = bad_of(j), next_bad = 0;
    rows.copy(pages.keys, next_row, place(0, 0));
    rows.copy(pages.values, next_row, place(0, 1));
    const auto copy_keys = [&](int j, int buffer) {
      advance(j);
      next_row = row_of(j);
      next_bad = bad_of(j);
      rows.copy(pages.keys, next_row, place(buffer, 0));
    };
    if (j + 1 < end) copy_keys(j + 1, 1);
    for (int buffer = 0; j < end; ++j, buffer ^= 1) {
      const bool more = j + 1 < end;
      if (more) wait_copies<2 * kCopies>();
      else wait_copies<kCopies>();
      block_sync();
      if (more) rows.copy(pages.values, next_row, place(buffer ^ 1, 1));
      tree_turn();
      const uint32_t now = bad;
      bad = next_bad;
      const auto middle = [&] {
        if (more) wait_copies<2 * kCopies>();
        else wait_copies<0>();
        const int left = rows_left(j, now);
        if (left < 16) TreeRows<D, false>::clear(place(buffer, 1), left, lane);
        block_sync();
        if (j + 2 < end) copy_keys(j + 2, buffer);
      };
      if (idle) middle();
      else compute(j, buffer, now, middle, TreeNothing());
    }
  } else {
    // the next unit is widened into LDS beside the products with V
    constexpr int kParts = TreeRows<D, true>::kParts, kSteps = D / 16;
    TreeRows<D, true> key, value;
    const auto load = [&](int j) {
      const int64_t row = row_of(j);
      key.load(pages.keys, pages.key_scales, row, lane);
      value.load(pages.values, pages.value_scales, row, lane);
    };
    const auto store = [&](int buffer, int n) {                // of 2 kParts
      if (n < kParts) key.store(place(buffer, 0), n, lane);
      else value.store(place(buffer, 1), n - kParts, lane);
    };
    load(j);
    uint32_t bad = bad_of(j);
    value.limit(rows_left(j, bad), lane);
#pragma unroll
    for (int n = 0; n < 2 * kParts; ++n) store(0, n);
    if (j + 1 < end) {
      advance(j + 1);
      load(j + 1);
    }
    for (int buffer = 0; j < end; ++j, buffer ^= 1) {
      block_sync();
      tree_turn();
      const uint32_t now = bad;
      if (j + 1 < end) {
        bad = bad_of(j + 1);
        const int left = rows_left(j + 1, bad);
        if (left < 16) value.limit(left, lane);
      }
      // (behind the last unit what is widened is not read)
      const auto widen = [&](int t) {
        if constexpr (2 * kParts >= kSteps) {
#pragma unroll
          for (int n = 0; n < 2 * kParts / kSteps; ++n) store(buffer ^ 1, t * (2 * kParts / kSteps) + n);
        }
      };
      static_assert(2 * kParts % kSteps == 0, "parts are dealt evenly");
      if (kCareful || idle) {
        if (!idle) compute(j, buffer, now, TreeNothing(), TreeNothing());
#pragma unroll
        for (int n = 0; n < 2 * kParts; ++n) store(buffer ^ 1, n);
      } else {
        compute(j, buffer, now, TreeNothing(), widen);
      }
      if (j + 2 < end) {
        advance(j + 2);
        load(j + 2);
      }
    }
  }
}

// WC waves side by side hold 32 columns each.
template <int D, bool kFour, int WC>
__global__ __launch_bounds__(kTreeThreads, TreeShape<D>::kPerCu) void paged_tree_kernel(TreeArgs a) {
  constexpr int WK = 4 / WC, kColumns = 32 * WC;
  __shared__ __align__(16) uint8_t tiles[2][2][TreeShape<D>::kTile];
  __shared__ int wrong[4];
  __shared__ float part_m[kColumns], part_l[kColumns];
  const int lane = threadIdx.x & 63, w = first_lane(threadIdx.x >> 6), half = lane >> 5;
  const int wc = w % WC, wk = w / WC;
  TreeScan scan;
  scan.load(a, kColumns, lane);
  int total = scan.total();
  for (int b0 = kWave; b0 < a.batch; b0 += kWave) {
    TreeScan more;
    more.load(a, kColumns, b0 + lane);
    total += more.total();
  }
  const TreeRun run(total, a.grid, a.inv_grid);
  const int begin = run.begin(blockIdx.x), end = run.begin(blockIdx.x + 1);
  TreeStream s;
  if (begin >= end || !s.find(a, kColumns, lane, scan, begin)) return;
  for (int u = begin;;) {
    const int j0 = u - s.first, j1 = min(end, s.first + s.x.units) - s.first;
    const int col = s.tile * kColumns + 32 * wc + (lane & 31);
    const int n = min(col, a.cols - 1);
    const int token = divide(n, a.group, a.inv_group);
    const int head = s.kvh * a.group + n - token * a.group;
    const bool idle = s.tile * kColumns + 32 * wc >= a.cols;
    u32x4 q[D / 16];
    const uint16_t* qr = a.q + s.b * a.qs_b + token * a.qs_t + head * a.qs_h + 8 * half;
    // Queries of padding may hold anything: 0, so that such columns are odd (below) only where others
    // are, from K and V.
    const uint32_t q_keep = token < s.x.live ? a.q_keep : 0;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      q[kk] = *reinterpret_cast<const u32x4*>(qr + 16 * kk);
#pragma unroll
      for (int e = 0; e < 4; ++e) q[kk][e] = (q[kk][e] & q_keep) ^ a.q_flip;
    }
    TreeState<D> st;
    const LdsBytes lds = (LdsBytes)&tiles[0][0][0];
    tree_run<D, kFour, WC, false>(st, a, s, q, token, idle, lds, j0, j1, w, lane);
    float sum = 0.0f;
#pragma unroll
    for (const auto& o : st.o)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum = __builtin_fmaf(o[r], 0.0f, sum);
    const bool odd = __any(sum != sum);
    if (lane == 0) wrong[w] = odd;
    block_sync();
    if (wrong[0] | wrong[1] | wrong[2] | wrong[3]) {
      block_sync();
      tree_run<D, kFour, WC, true>(st, a, s, q, token, idle, lds, j0, j1, w, lane);
      block_sync();
    }
    st.l = other_half_sum(st.l);
    const float top = st.m == -INFINITY ? -INFINITY : st.m * a.scale_log2;
    st.m = top;
    if constexpr (WK == 2) {             // the second wave's part through LDS
      f32x4* held = reinterpret_cast<f32x4*>(&tiles[0][0][0]) + wc * (D / 4 * 32);
      if (wk == 1) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            held[(8 * i + 2 * r + half) * 32 + (lane & 31)] =
                f32x4{st.o[i][4 * r], st.o[i][4 * r + 1], st.o[i][4 * r + 2], st.o[i][4 * r + 3]};
        if (half == 0) {
          part_m[32 * wc + lane] = st.m;
          part_l[32 * wc + lane] = st.l;
        }
      }
      block_sync();
      if (wk == 0) {
        const float m1 = part_m[32 * wc + (lane & 31)], l1 = part_l[32 * wc + (lane & 31)];
        const float both = fmaxf(st.m, m1);
        const float w0 = st.m == -INFINITY ? 0.0f : exp2_fast(st.m - both);
        const float w1 = m1 == -INFINITY ? 0.0f : exp2_fast(m1 - both);
        st.m = both;
        st.l = w0 * st.l + w1 * l1;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const f32x4 x = held[(8 * i + 2 * r + half) * 32 + (lane & 31)];
#pragma unroll
            for (int y = 0; y < 4; ++y) st.o[i][4 * r + y] = w0 * st.o[i][4 * r + y] + w1 * x[y];
          }
      }
    }
    const bool whole = j0 == 0 && j1 == s.x.units;
    const int slot = 2 * blockIdx.x + (u == begin ? 0 : 1);
    if (j0 == 0 && threadIdx.x == 0) {
      const int parts = whole ? 1 : run.owner(s.first + s.x.units - 1) - blockIdx.x + 1;
      a.parts[((int64_t)s.b * a.kv_heads + s.kvh) * a.col_tiles + s.tile] =
          u32x2{(uint32_t)slot, (uint32_t)parts};
    }
    if (wk == 0 && col < a.cols && token < s.x.live) {
      if (whole) {
        const int64_t row = ((int64_t)s.b * a.tokens + token) * a.q_heads + head;
        const float inv = st.m == -INFINITY && st.l == 0.0f ? 0.0f : 1.0f / st.l;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int r = 0; r < 16; r += 4)
            *reinterpret_cast<u32x2*>(a.out + row * D + 32 * i + mfma32_row(r, lane)) =
                u32x2{pack_bf16x2(st.o[i][r] * inv, st.o[i][r + 1] * inv),
                      pack_bf16x2(st.o[i][r + 2] * inv, st.o[i][r + 3] * inv)};
        if (half == 0 && a.lse) a.lse[row] = (st.m + __builtin_amdgcn_logf(st.l)) * kLn2;
      } else {
        const int c = 32 * wc + (lane & 31);
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            *reinterpret_cast<f32x4*>(
                a.part_o + (((int64_t)slot * (D / 4) + 8 * i + 2 * r + half) * kColumns + c) * 4) =
                f32x4{st.o[i][4 * r], st.o[i][4 * r + 1], st.o[i][4 * r + 2], st.o[i][4 * r + 3]};
        if (half == 0) {
          a.part_ml[((int64_t)slot * kColumns + c) * 2] = st.m;
          a.part_ml[((int64_t)slot * kColumns + c) * 2 + 1] = st.l;
        }
      }
    }
    u = s.first + j1;
    if (u >= end || !s.next(a, kColumns)) return;
    block_sync();                        // LDS is read before it is written again
  }
}

// ------------------------------------------------------------------------ merge
//
// An item is eight columns of a stream by 32 dims; W waves take its partials in turn. Columns of one
// workgroup are written already, columns of tokens that are not live are written here.
template <int D, int W, int kColumns>
__global__ __launch_bounds__(64 * (W == 1 ? 4 : W)) void paged_tree_merge_kernel(TreeArgs a, int groups,
                                                                                int64_t items) {
  constexpr int kItems = W == 1 ? 4 : 1, kAtOnce = W == 1 ? 4 : 8;
  __shared__ float red_m[W][8], red_l[W][8];
  __shared__ __align__(16) f32x4 red_o[W][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c8 = lane & 7, q8 = lane >> 3;
  for (int64_t at = (int64_t)blockIdx.x * kItems; at < items; at += (int64_t)gridDim.x * kItems) {
    const int64_t item = at + (W == 1 ? w : 0);
    if (item >= items) return;           // W == 1: waves on their own
    const int dims = (int)(item % (D / 32));
    const int64_t rest = item / (D / 32);
    const int group = (int)(rest % groups);
    const int64_t bh = rest / groups;
    const int kvh = (int)(bh % a.kv_heads), b = (int)(bh / a.kv_heads);
    const int col = 8 * group + c8, n = min(col, a.cols - 1);
    const int token = divide(n, a.group, a.inv_group);
    const int head = kvh * a.group + n - token * a.group;
    const int64_t row = ((int64_t)b * a.tokens + token) * a.q_heads + head;
    const int dim = 32 * dims + 4 * q8;
    TreeLengths x;
    x.of(a, kColumns, a.map.starts[b], a.map.counts ? a.map.counts[b] : a.tokens);
    const bool dead = token >= x.live, mine = col < a.cols;
    if (dead && mine && (W == 1 || w == 0)) {
      *reinterpret_cast<u32x2*>(a.out + row * D + dim) = u32x2{};
      if (dim == 0 && a.lse) a.lse[row] = -INFINITY;
    }
    const int tile = 8 * group / kColumns, c = 8 * group % kColumns + c8;
    int slot0 = 0, parts = 0;
    if (tile < x.tiles) {
      const u32x2 held = a.parts[bh * a.col_tiles + tile];
      slot0 = (int)min(held[0], 2u * a.grid - 1);               // in bounds whatever it holds
      parts = min((int)held[1], a.grid - slot0 / 2);
    }
    if (parts <= 1) continue;            // the same for the whole workgroup
    // the stream is the first one of every workgroup but perhaps the first
    const auto slot = [&](int y) { return y == 0 ? slot0 : (slot0 & ~1) + 2 * y; };
    float top = -INFINITY, sum = 0.0f;
    f32x4 acc{};
    for (int y0 = w % W; y0 < parts; y0 += W * kAtOnce) {
      f32x4 po[kAtOnce];
      float m[kAtOnce], l[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const int y = min(y0 + W * k, parts - 1);
        const float* ml = a.part_ml + ((int64_t)slot(y) * kColumns + c) * 2;
        po[k] = *reinterpret_cast<const f32x4*>(
            a.part_o + (((int64_t)slot(y) * (D / 4) + dim / 4) * kColumns + c) * 4);
        const bool here = y0 + W * k < parts;
        m[k] = here ? ml[0] : -INFINITY;
        l[k] = here ? ml[1] : 0.0f;
        if (!here) po[k] = f32x4{};
      }
      float higher = top;
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) higher = fmaxf(higher, m[k]);
      const float old = top == -INFINITY ? 0.0f : exp2_fast(top - higher);
      sum *= old;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] *= old;
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        // 0 where it saw nothing; a NaN sum stays NaN
        const float wt = m[k] == -INFINITY ? 0.0f : exp2_fast(m[k] - higher);
        sum += wt * l[k];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += wt * po[k][e];
      }
      top = higher;
    }
    if constexpr (W > 1) {
      if (q8 == 0) {
        red_m[w][c8] = top;
        red_l[w][c8] = sum;
      }
      red_o[w][lane] = acc;
      block_sync();
      float all = -INFINITY;
#pragma unroll
      for (int y = 0; y < W; ++y) all = fmaxf(all, red_m[y][c8]);
      sum = 0.0f;
      acc = f32x4{};
#pragma unroll
      for (int y = 0; y < W; ++y) {
        const float m = red_m[y][c8], wt = m == -INFINITY ? 0.0f : exp2_fast(m - all);
        sum += wt * red_l[y][c8];
        const f32x4 o = red_o[y][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += wt * o[e];
      }
      top = all;
      block_sync();
    }
    if (dead || !mine || (W > 1 && w != 0)) continue;
    const float inv = top == -INFINITY && sum == 0.0f ? 0.0f : 1.0f / sum;
    *reinterpret_cast<u32x2*>(a.out + row * D + dim) =
        u32x2{pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv)};
    if (dim == 0 && a.lse) a.lse[row] = (top + __builtin_amdgcn_logf(sum)) * kLn2;
  }
}

// ------------------------------------------------------------------------- plan

// Depths and ancestor masks from parents, one workgroup per sequence: after step s a node's mask
// holds its nearest 2^s ancestors and itself, and `up` is the one 2^s further up.
__global__ __launch_bounds__(kTreeMaxTokens) void draft_tree_kernel(const int32_t* parents, int tokens,
                                                                    int words, int32_t* depths,
                                                                    uint64_t* masks) {
  constexpr int kWords = kTreeMaxTokens / 64;
  __shared__ uint64_t mask[kTreeMaxTokens][kWords];
  __shared__ int up[kTreeMaxTokens];
  const int i = threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * tokens + i;
  int mine = -1;
  uint64_t seen[kWords] = {};
  if (i < tokens) {
    mine = parents[row];
    if (mine >= i || mine < 0) mine = -1;
#pragma unroll
    for (int w = 0; w < kWords; ++w) seen[w] = w == i / 64 ? 1ull << (i % 64) : 0;
  }
  for (int reach = 1; reach < tokens; reach *= 2) {
    up[i] = mine;
#pragma unroll
    for (int w = 0; w < kWords; ++w) mask[i][w] = seen[w];
    block_sync();
    if (mine >= 0) {
#pragma unroll
      for (int w = 0; w < kWords; ++w) seen[w] |= mask[mine][w];
      mine = up[mine];
    }
    block_sync();
  }
  if (i >= tokens) return;
  int depth = -1;
#pragma unroll
  for (int w = 0; w < kWords; ++w) {
    depth += __popcll(seen[w]);
    if (w < words) masks[row * words + w] = seen[w];
  }
  depths[row] = depth;
}

// ------------------------------------------------------------------------- host

struct TreeSizes {
  int64_t keys, streams, rows;
  int columns;                           // of a tile
};

static bool tree_sizes(const spx_paged_cache& z, int q_heads, int max_keys, TreeSizes& s) {
  if (z.table_width <= 0 || z.page_size <= 0 || max_keys < 0 || z.batch <= 0 || z.tokens <= 0 ||
      z.tokens > kTreeMaxTokens || q_heads <= 0 || q_heads > 1 << 20 || z.kv_heads <= 0 ||
      q_heads % z.kv_heads != 0)
    return false;
  if ((double)z.batch * z.tokens * q_heads > 0x7fffffff) return false;
  s.rows = (int64_t)z.batch * z.tokens * q_heads;
  s.keys = (int64_t)z.table_width * z.page_size;
  const int64_t cols = (int64_t)z.tokens * (q_heads / z.kv_heads);
  s.columns = cols <= 64 ? 64 : 128;
  s.streams = (int64_t)z.batch * z.kv_heads * ((cols + s.columns - 1) / s.columns);
  // units are counted in 32 bits, also where max_keys is no bound after all
  if ((s.keys + kTreeKeys - 1) / kTreeKeys > 0x7fffffff / s.streams) return false;
  if (max_keys > 0) s.keys = std::min<int64_t>(s.keys, max_keys);
  return true;
}

static int tree_grid(const TreeSizes& s, int head_dim) {
  const int most = kTreeCus * (head_dim == 128 ? TreeShape<128>::kPerCu : TreeShape<256>::kPerCu);
  return (int)std::min<int64_t>(most, s.streams * ((s.keys + kTreeKeys - 1) / kTreeKeys));
}

// Rows from which on a wave joins each item's partials by itself, and partials of a stream from which
// on 16 waves do: 128 of 64 columns (56 in use) 6.6 us instead of 13.4 with four waves, 32 of 128
// columns 19.2 instead of 9.0.
constexpr int kTreeWaveRows = 2048, kTreeManyParts = 64;

template <int D, bool kFour, int WC>
static int launch_tree(TreeArgs a, const TreeSizes& z, hipStream_t st) {
  constexpr int kColumns = 32 * WC;
  paged_tree_kernel<D, kFour, WC><<<(unsigned)a.grid, kTreeThreads, 0, st>>>(a);
  const int groups = (a.cols + 7) / 8;
  const int64_t items = (int64_t)a.batch * a.kv_heads * groups * (D / 32);
  const auto grid = [](int64_t n) { return (unsigned)std::min<int64_t>(n, 1 << 20); };
  if (z.rows >= kTreeWaveRows)
    paged_tree_merge_kernel<D, 1, kColumns><<<grid((items + 3) / 4), 256, 0, st>>>(a, groups, items);
  else if (a.grid >= kTreeManyParts * z.streams)
    paged_tree_merge_kernel<D, 16, kColumns><<<grid(items), 1024, 0, st>>>(a, groups, items);
  else
    paged_tree_merge_kernel<D, 4, kColumns><<<grid(items), 256, 0, st>>>(a, groups, items);
  return launch_status("paged_tree_attention");
}

template <int D, bool kFour>
static int launch_tree(const TreeArgs& a, const TreeSizes& z, hipStream_t st) {
  return z.columns == 64 ? launch_tree<D, kFour, 2>(a, z, st) : launch_tree<D, kFour, 4>(a, z, st);
}

}  // namespace spx

using namespace spx;

extern "C" int spx_draft_tree(const int32_t* parents, int batch, int tokens, int32_t* depths,
                              uint64_t* masks, void* stream) {
  SPX_REQUIRE(parents && depths && masks, SPX_EINVAL, "null pointer");
  SPX_REQUIRE(batch > 0 && tokens > 0 && tokens <= kTreeMaxTokens, SPX_EINVAL,
              "bad shape: batch %d tokens %d (at most %d tokens)", batch, tokens, kTreeMaxTokens);
  SPX_REQUIRE(batch <= 1 << 23, SPX_EINVAL, "%d sequences are more than 2^23", batch);
  SPX_REQUIRE(((reinterpret_cast<uintptr_t>(parents) | reinterpret_cast<uintptr_t>(depths)) & 3) == 0 &&
                  (reinterpret_cast<uintptr_t>(masks) & 7) == 0,
              SPX_EINVAL, "parents and depths must be 4-byte, masks 8-byte aligned");
  draft_tree_kernel<<<(unsigned)batch, kTreeMaxTokens, 0, static_cast<hipStream_t>(stream)>>>(
      parents, tokens, (tokens + 63) / 64, depths, masks);
  return launch_status("draft_tree");
}

extern "C" int64_t spx_paged_tree_attention_workspace_bytes(const spx_paged_cache* cache, int q_heads,
                                                            int max_keys) {
  TreeSizes z;
  if (cache == nullptr || (cache->head_dim != 128 && cache->head_dim != 256) ||
      !tree_sizes(*cache, q_heads, max_keys, z))
    return -1;
  const int64_t grid = tree_grid(z, cache->head_dim);
  return 2 * grid * z.columns * (cache->head_dim + 2) * 4 + z.streams * 8;
}

extern "C" int spx_paged_tree_attention(const spx_paged_cache* cache, const void* q,
                                        const int64_t* q_strides, int q_heads, const uint64_t* masks,
                                        int max_keys, float scale, void* workspace, void* out,
                                        float* lse, void* stream) {
  TreeArgs a{};
  const int status = paged_map(a.map, cache);
  if (status != SPX_OK) return status;
  TreeSizes z;
  SPX_REQUIRE(tree_sizes(*cache, q_heads, max_keys, z), SPX_EINVAL,
              "bad shape: batch %d tokens %d (at most %d) q_heads %d kv_heads %d max_keys %d",
              cache->batch, cache->tokens, kTreeMaxTokens, q_heads, cache->kv_heads, max_keys);
  SPX_REQUIRE(q && q_strides && out && masks && workspace, SPX_EINVAL, "null pointer");
  SPX_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) |
                reinterpret_cast<uintptr_t>(workspace)) & 15) == 0 &&
                  q_strides[3] == 1 && ((q_strides[0] | q_strides[1] | q_strides[2]) & 7) == 0,
              SPX_EINVAL,
              "q, out, workspace: bases must be 16-byte aligned, q's dim stride 1, the others "
              "multiples of 8");
  SPX_REQUIRE((reinterpret_cast<uintptr_t>(masks) & 7) == 0, SPX_EINVAL,
              "masks must be 8-byte aligned");
  const bool four = cache->key_scales != nullptr;
  a.q = static_cast<const uint16_t*>(q);
  a.qs_b = q_strides[0]; a.qs_t = q_strides[1]; a.qs_h = q_strides[2];
  a.key_pages = cache->key_pages; a.value_pages = cache->value_pages;
  a.key_scales = static_cast<const uint8_t*>(cache->key_scales);
  a.value_scales = static_cast<const uint8_t*>(cache->value_scales);
  a.masks = masks;
  a.words = (cache->tokens + 63) / 64;
  a.batch = cache->batch; a.tokens = cache->tokens;
  a.q_heads = q_heads; a.kv_heads = cache->kv_heads; a.group = q_heads / cache->kv_heads;
  a.cols = cache->tokens * a.group;
  a.col_tiles = (a.cols + z.columns - 1) / z.columns;
  a.grid = tree_grid(z, cache->head_dim);
  a.inv_grid = 1.0 / a.grid;
  a.inv_group = 1.0 / a.group;
  a.scale_log2 = scale == 0 ? 1.0f : (float)(std::abs((double)scale) * 1.4426950408889634);
  a.q_keep = scale == 0 ? 0 : 0xffffffffu;
  a.q_flip = scale < 0 ? 0x80008000u : 0;
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + (int64_t)2 * a.grid * z.columns * cache->head_dim;
  a.parts = reinterpret_cast<u32x2*>(a.part_ml + (int64_t)2 * a.grid * z.columns * 2);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (cache->head_dim == 128)
    return four ? launch_tree<128, true>(a, z, st) : launch_tree<128, false>(a, z, st);
  return four ? launch_tree<256, true>(a, z, st) : launch_tree<256, false>(a, z, st);
}
