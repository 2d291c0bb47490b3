// Attention weight that cached tokens gather: with the LSE of an attention call over the paged cache,
//
//   weights[b, kvh, p] += sum over rows (i, h of the group) that see p of exp(scale q k_p - lse).
//
// Columns n = i group + h of a KV head, 16 to a matrix tile. v_mfma_f32_16x16x32_bf16 with Q as A and
// K as B operand: the scores of a key lie in one lane's four registers, so the sum over columns is
// in the lane but for the four lane groups at the end. K comes straight from the pages into registers.
//
// With s and L the scale and the LSE in units of log 2, each rounded once (s', L'), a weight is
//   2^(s x - L) = 2^(s' x - L') 2^e,   e = (s - s') x - (L - L') = (s / s' - 1) L' - (L - L') nearly,
// as s' x is L' where the weight counts: the columns' factor 2^e makes up for both roundings.
//
// Two kernels. Up to 16 columns (decode steps) a wave has Q in registers and walks the keys by itself, the
// next 32 or 64 under way: bound by the pages' bytes (64 sequences of up to 8192 keys in 4 bits, 32/8
// heads: 34 us, 5.0 TB/s). Else a wave holds 64 keys in registers and walks the columns, which the
// workgroup copies into LDS a unit ahead: bound by three vector instructions a score and the products,
// which overlap little (2000 tokens over 16000 keys, 28/4 heads: 243 us a call with the join, 0.88
// PFLOP/s, matrix units busy 46 % of the cycles; scores of one tile spread over the products of the next
// by hand: 265 for 256). At D = 128 that kernel spills 10 (bf16) or 11 registers (4 bits).
#include <algorithm>
#include <cmath>

#include "paged_tiles.h"

namespace spx {

// Up to kPwFewCols columns the first kernel: a batch of 16 x 8000 keys in 4 bits, 32/8 heads, 4 tokens
// 18 us (30 with the second); 4 x 8000, D = 256, bf16 14.7 (16.8).
constexpr int kPwFewCols = 16;
// Up to kPwWholeCols columns a block of keys has one workgroup of 4 waves and no partial sums: 64 tokens
// over 32640 keys, 28/4 heads 28 us (32 + 5 shared by workgroups of 8 waves), 8 x 16 over 4000, 32/8 heads
// 16 (23 + 5). Beyond, runs of columns are shared: 301 tokens over 8000, 32/8 heads 36 + 5 us (53 by
// whole blocks).
constexpr int kPwWholeCols = 512;
constexpr int kPwCus = 256;
constexpr int kPwTiles = 4;              // of 16 keys, a wave's

// W waves of a workgroup: each has 64 keys and brings in 16 columns of a unit.
constexpr int kPwWaves = 4, kPwManyWaves = 8;
__host__ __device__ constexpr int weight_keys(int waves) { return 16 * kPwTiles * waves; }
__host__ __device__ constexpr int weight_cols(int waves) { return 16 * waves; }

typedef int i32x4 __attribute__((ext_vector_type(4)));

// Tiles of 16 keys that a wave has under way for few columns, and waves per SIMD. (bf16, D = 128 with 4
// and 2 in place of 2 and 4: 100000 keys, 32/8 heads 44.4 us, not 42.8; 2000 keys 5.4, not 4.4.)
template <bool kFour>
constexpr int kPwFewTiles = kFour ? 4 : 2;
template <int D>
constexpr int kPwFewPerSimd = D == 128 ? 4 : 2;

struct PagedWeightArgs {
  PagedMap map;
  const uint16_t* q;
  int64_t qs_b, qs_t, qs_h;
  const float* lse;                      // [B, T, Hq]
  const void* key_pages;
  const void* value_pages;               // (not read)
  const uint8_t* key_scales;
  const uint8_t* value_scales;
  int batch, tokens, q_heads, kv_heads, group;
  int blocks;                            // blocks of keys that the table reaches
  int whole;                             // blocks are not shared by workgroups
  int grid;                              // workgroups, or waves, that share the work
  double inv_grid, inv_group;
  float scale, scale_rest;               // scale log2(e), rounded; what of it is missing, relative
  float* weights;                        // [B, Hkv, row]
  int64_t row;
  float* part;                           // [2 grid][keys of a block]
  u32x2* parts;                          // [B, Hkv, blocks]
};

struct WeightLengths {
  int start, live, keys, blocks, chunks;
  __device__ __forceinline__ void of(const PagedWeightArgs& a, int block, int cols, int start_,
                                     int count) {
    start = start_;
    const int64_t room = a.map.capacity() - start;
    live = start < 0 ? 0
                     : max(0, min(min(count, a.tokens), (int)min(room, (int64_t)a.tokens)));
    keys = live > 0 ? start + live : 0;
    blocks = (keys + block - 1) / block;
    chunks = (live * a.group + cols - 1) / cols;
  }
  __device__ __forceinline__ void load(const PagedWeightArgs& a, int block, int cols, int b) {
    of(a, block, cols, scalar_load(a.map.starts + b),
       a.map.counts ? scalar_load(a.map.counts + b) : a.tokens);
  }
};

// What is dealt to the workgroups: chunks of columns of the blocks of keys, or whole blocks.
struct WeightScan {                      // of 64 sequences, one a lane
  int units, sum;
  __device__ __forceinline__ void load(const PagedWeightArgs& a, int block, int cols, int b) {
    WeightLengths x;
    int start = -1, count = a.tokens;
    if (b < a.batch) {
      start = a.map.starts[b];
      if (a.map.counts) count = a.map.counts[b];
    }
    x.of(a, block, cols, start, count);
    units = x.chunks == 0 ? 0 : x.blocks * (a.whole ? 1 : x.chunks) * a.kv_heads;
    sum = wave_prefix(units);
  }
  __device__ __forceinline__ int total() const { return __builtin_amdgcn_readlane(sum, kWave - 1); }
};

struct WeightUnit {
  WeightLengths x;
  int b, kvh, at, chunk;                 // at: which of the blocks, in the order of the runs

  __device__ __forceinline__ bool find(const PagedWeightArgs& a, int block, int cols, int lane,
                                       WeightScan scan, int u) {
    int before = 0, b0 = 0;
    uint64_t past;
    while (!(past = __ballot(before + scan.sum > u))) {
      before += scan.total();
      b0 += kWave;
      if (b0 >= a.batch) return false;
      scan.load(a, block, cols, b0 + lane);
    }
    const int l = __builtin_ctzll(past);
    b = b0 + l;
    before += __builtin_amdgcn_readlane(scan.sum - scan.units, l);
    x.load(a, block, cols, b);
    if (x.blocks <= 0 || x.chunks <= 0 || u < before) return false;
    const int each = a.whole ? 1 : x.chunks;
    const int stream = (u - before) / each;
    chunk = u - before - stream * each;
    kvh = stream / x.blocks;
    at = stream - kvh * x.blocks;
    return kvh < a.kv_heads;
  }
  __device__ __forceinline__ bool next(const PagedWeightArgs& a, int block, int cols) {
    if (++chunk < x.chunks) return true;
    chunk = 0;
    if (++at < x.blocks) return true;
    at = 0;
    if (++kvh < a.kv_heads) return true;
    kvh = 0;
    do {
      if (++b >= a.batch) return false;
      x.load(a, block, cols, b);
    } while (x.blocks == 0 || x.chunks == 0);
    return true;
  }
  // First and last in turn: with several chunks the late ones of a prompt's blocks are seen by few
  // columns, and so every run has its share of them.
  __device__ __forceinline__ int block() const {
    return x.chunks == 1 ? at : at % 2 ? x.blocks - 1 - at / 2 : at / 2;
  }
};

struct WeightRun {
  int per, rest;
  __device__ __forceinline__ WeightRun(int total, int grid, double inv)
      : per(first_lane(divide(total, grid, inv))), rest(total - per * grid) {}
  __device__ __forceinline__ int begin(int w) const { return w * per + min(w, rest); }
  __device__ __forceinline__ int owner(int u) const {
    const int wide = rest * (per + 1);
    return u < wide ? u / (per + 1) : rest + (u - wide) / max(per, 1);
  }
};

// A column's LSE in units of log 2, rounded, the factor that makes up for the roundings, and the last
// key that it sees (-1: none).
struct WeightColumn {
  float hi, factor;
  int last;
  __device__ __forceinline__ WeightColumn(const PagedWeightArgs& a, float lse, int last_key) {
    hi = lse * kLog2e;
    // log2(e) is kLog2e + 1.925963033500e-8
    const float lo = __builtin_fmaf(lse, kLog2e, -hi) + lse * 1.925963033500e-8f;
    // (finite whatever the LSE is: it multiplies zeros too)
    const float e = __builtin_fmaf(hi, a.scale_rest, -lo);
    factor = __builtin_fabsf(e) < 1.0f ? exp2_fast(e) : 1.0f;
    last = lse == -INFINITY ? -1 : last_key;
  }
};

// Sums over the four lane groups: tile g's in group g (of two tiles: g / 2's).
__device__ __forceinline__ float weight_sums(const float (&x)[4]) {
  float y[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[i]), __float_as_uint(x[i + 2]),
                                                    false, false);
    y[i] = __uint_as_float(h[0]) + __uint_as_float(h[1]);
  }
  const auto h = __builtin_amdgcn_permlane16_swap(__float_as_uint(y[0]), __float_as_uint(y[1]), false,
                                                  false);
  return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}
__device__ __forceinline__ float weight_sums(const float (&x)[2]) {
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[0]), __float_as_uint(x[1]), false,
                                                  false);
  const float y = __uint_as_float(h[0]) + __uint_as_float(h[1]);
  return y + __shfl_xor(y, 16);
}

// ------------------------------------------------------------------ few columns

template <int D, bool kFour>
__global__ __launch_bounds__(64 * kPwWaves, kPwFewPerSimd<D>) void
paged_weight_few_kernel(PagedWeightArgs a) {
  constexpr int T = kPwFewTiles<kFour>, kKeys = 16 * T, KK = D / 32;
  const int lane = threadIdx.x & 63, w = first_lane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  WeightScan scan;
  scan.load(a, kKeys, kPwFewCols, lane);
  int total = scan.total();
  for (int b0 = kWave; b0 < a.batch; b0 += kWave) {
    WeightScan more;
    more.load(a, kKeys, kPwFewCols, b0 + lane);
    total += more.total();
  }
  const WeightRun run(total, a.grid, a.inv_grid);
  const int wave = blockIdx.x * kPwWaves + w;
  int u = run.begin(wave);
  const int end = run.begin(wave + 1);
  WeightUnit s, next;                    // unit u and u + 1
  if (u >= end || !s.find(a, kKeys, kPwFewCols, lane, scan, u)) return;
  // lane t: page of tile t % T
  const auto fetch_ids = [&](const WeightUnit& s) {
    const int64_t p = (int64_t)s.at * kKeys + lane % T * 16;
    return a.map.page(s.b, (int)min(p, (int64_t)s.x.keys - 1));
  };
  struct Keys {
    KeyTile<D, kFour> tile[T];
    float old;                           // the lane's key: its weight
    float* at;                           // and where it stands, null: nowhere
  };
  const int mine = T == 4 ? g : g >> 1;  // the lane's tile at the end
  const auto load = [&](Keys& k, const WeightUnit& s, int ids) {
    const HeadPages<D, kFour> pages(a, s.kvh);
    const int key0 = s.at * kKeys;
#pragma unroll
    for (int t = 0; t < T; ++t)
      k.tile[t].load(pages, pages.row(max(__builtin_amdgcn_readlane(ids, t), 0), key0 + 16 * t), c, g);
    const uint64_t lost = __ballot(ids < 0);
    const int p = key0 + 16 * mine + c;
    const bool stands = p < s.x.keys && !(lost >> mine & 1) && (T == 4 || g % 2 == 0);
    k.at = stands ? a.weights + ((int64_t)s.b * a.kv_heads + s.kvh) * a.row + p : nullptr;
    k.old = stands ? *k.at : 0.0f;
  };
  u32x4 q[KK];
  float hi[4], factor[4];
  int last[4];
  int held_b = -1, held_kvh = 0;
  int ids = fetch_ids(s);
  const auto step = [&](Keys& now, Keys& coming) {
    const WeightUnit at = s;
    if (at.b != held_b || at.kvh != held_kvh) {
      held_b = at.b;
      held_kvh = at.kvh;
      const int live = at.x.live * a.group;
      const auto place = [&](int n, int& token, int& head) {
        n = min(n, live - 1);
        token = divide(n, a.group, a.inv_group);
        head = at.kvh * a.group + n - token * a.group;
      };
      int token, head;
      place(c, token, head);
      const uint16_t* row = a.q + at.b * a.qs_b + token * a.qs_t + head * a.qs_h;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        q[kk] = *reinterpret_cast<const u32x4*>(row + KeyTile<D, kFour>::dim(kk, g));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        place(4 * g + r, token, head);
        const WeightColumn x(a, a.lse[((int64_t)at.b * a.tokens + token) * a.q_heads + head],
                             4 * g + r < live ? at.x.start + token : -1);
        hi[r] = x.hi;
        factor[r] = x.factor;
        last[r] = x.last;
      }
    }
    const bool more = ++u < end && next.next(a, kKeys, kPwFewCols);
    if (more) {
      load(coming, next, ids);
      s = next;
    }
    if (more && u + 1 < end) {
      WeightUnit after = next;
      if (after.next(a, kKeys, kPwFewCols)) ids = fetch_ids(after);
    }
    const int key0 = at.at * kKeys + c;
    float acc[T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
      f32x4 x{};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) x = mfma16(q[kk], now.tile[t].operand(kk, g), x);
      acc[t] = 0.0f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = exp2_fast(__builtin_fmaf(x[r], a.scale, -hi[r]));
        acc[t] = __builtin_fmaf(key0 + 16 * t <= last[r] ? p : 0.0f, factor[r], acc[t]);
      }
    }
    const float sum = weight_sums(acc);
    if (now.at) *now.at = now.old + sum;
    return more;
  };
  Keys one, two;
  load(one, s, ids);
  next = s;
  if (u + 1 < end) {
    WeightUnit after = next;
    if (after.next(a, kKeys, kPwFewCols)) ids = fetch_ids(after);
  }
  while (step(one, two) && step(two, one)) {}
}

// ----------------------------------------------------------------- many columns

// Four times 16 bytes a lane from from[i] to to + 1024 i + 16 lane, past the registers.
__device__ __forceinline__ void copy_rows_to_lds(const uint64_t (&from)[4], LdsBytes to) {
#if defined(__HIP_DEVICE_COMPILE__)
  const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)to);
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %2, off\n\t"
      "s_add_u32 m0, m0, 0x400\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %3, off\n\t"
      "s_add_u32 m0, m0, 0x400\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %4, off\n\t"
      "s_add_u32 m0, m0, 0x400\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %5, off\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "s"(m0), "v"(from[0]), "v"(from[1]), "v"(from[2]), "v"(from[3])
      : "memory", "scc");
#endif
}

// A unit's columns in LDS: rows of Q, 16-byte chunks exchanged within a row by an XOR with row % 16.
template <int D, int W>
struct WeightColumns {
  static constexpr int kLanes = D / 8, kRows = kWave / kLanes, kCopies = 16 / kRows;
  static constexpr int kCols = weight_cols(W);
  uint16_t q[kCols * D];
  float hi[kCols], factor[kCols];
  int last[kCols];
  int least[W], most[W];                 // of 16 columns: keys up to it are seen by all, behind it by none
};

template <int D, bool kFour, int W>
__global__ __launch_bounds__(64 * W, D == 128 ? (W == kPwWaves ? 3 : 4) : 2) void
paged_weight_kernel(PagedWeightArgs a) {
  constexpr int T = kPwTiles, KK = D / 32, kKeys = weight_keys(W), kCols = weight_cols(W);
  using Columns = WeightColumns<D, W>;
  __shared__ __align__(16) Columns columns[2];
  const int lane = threadIdx.x & 63, w = first_lane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  WeightScan scan;
  scan.load(a, kKeys, kCols, lane);
  int total = scan.total();
  for (int b0 = kWave; b0 < a.batch; b0 += kWave) {
    WeightScan more;
    more.load(a, kKeys, kCols, b0 + lane);
    total += more.total();
  }
  const WeightRun run(total, a.grid, a.inv_grid);
  const int begin = run.begin(blockIdx.x), end = run.begin(blockIdx.x + 1);
  WeightUnit s;
  if (begin >= end || !s.find(a, kKeys, kCols, lane, scan, begin)) return;
  // A wave brings 16 columns in; finish() after the copies are there.
  float lse = 0.0f;
  int last_key = 0, latest = 0;
  const auto stage = [&](const WeightUnit& s, Columns& to) {
    const int n = s.chunk * kCols + 16 * w + c, m = min(n, s.x.live * a.group - 1);
    const int token = divide(m, a.group, a.inv_group), head = s.kvh * a.group + m - token * a.group;
    const uint64_t row = (uint64_t)(a.q + s.b * a.qs_b + token * a.qs_t + head * a.qs_h);
    lse = a.lse[((int64_t)s.b * a.tokens + token) * a.q_heads + head];
    last_key = n == m ? s.x.start + token : -1;
    latest = s.x.start + __builtin_amdgcn_readlane(token, 15);
    const LdsBytes place = (LdsBytes)to.q + 16 * w * 2 * D;
#pragma unroll
    for (int i = 0; i < Columns::kCopies; i += 4) {
      uint64_t from[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = Columns::kRows * (i + j) + lane / Columns::kLanes;
        from[j] = ((uint64_t)(uint32_t)__shfl((int)(row >> 32), r) << 32 |
                   (uint32_t)__shfl((int)row, r)) +
                  ((lane % Columns::kLanes) ^ r) * 16;
      }
      copy_rows_to_lds(from, place + 1024 * i);
    }
  };
  const auto finish = [&](Columns& to) {
    const WeightColumn x(a, lse, last_key);
    const bool dead = __any(x.last < 0);
    if (lane < 16) {
      to.hi[16 * w + lane] = x.hi;
      to.factor[16 * w + lane] = x.factor;
      to.last[16 * w + lane] = x.last;
    }
    if (lane == 0) {
      to.least[w] = dead ? -1 : last_key;
      to.most[w] = latest;
    }
    wait_copies<0>();
  };
  u32x4 key[T][KK];
  bool placed = false;                   // the lane's key of tile g
  const auto load_keys = [&](const WeightUnit& s) {
    const HeadPages<D, kFour> pages(a, s.kvh);
    const int key0 = s.block() * kKeys + w * 16 * T;
    const int64_t p = (int64_t)key0 + lane % T * 16;
    const int ids = a.map.page(s.b, (int)min(p, (int64_t)s.x.keys - 1));
    KeyTile<D, kFour> tile[T];
#pragma unroll
    for (int t = 0; t < T; ++t)
      tile[t].load(pages, pages.row(max(__builtin_amdgcn_readlane(ids, t), 0), key0 + 16 * t), c, g);
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) key[t][kk] = tile[t].operand(kk, g);
    placed = !(__ballot(ids < 0) >> g & 1);
  };
  float acc[T] = {};
  const auto compute = [&](const Columns& q, int key0, int ct, bool masked) {
    const LdsBytes row = (LdsBytes)q.q + (16 * ct + c) * 2 * D;
    f32x4 x[T];
#pragma unroll
    for (int t = 0; t < T; ++t) x[t] = f32x4{};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int piece = KeyTile<D, kFour>::dim(kk, g) / 8;
      const u32x4 qk = lds_load<u32x4>(row, (piece ^ c) << 4);
#pragma unroll
      for (int t = 0; t < T; ++t) x[t] = mfma16(qk, key[t][kk], x[t]);
    }
    const f32x4 hi = *reinterpret_cast<const f32x4*>(q.hi + 16 * ct + 4 * g);
    const f32x4 factor = *reinterpret_cast<const f32x4*>(q.factor + 16 * ct + 4 * g);
    i32x4 last{};
    if (masked) last = *reinterpret_cast<const i32x4*>(q.last + 16 * ct + 4 * g);
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float p = exp2_fast(__builtin_fmaf(x[t][r], a.scale, -hi[r]));
        if (masked) p = key0 + 16 * t + c <= last[r] ? p : 0.0f;
        acc[t] = __builtin_fmaf(p, factor[r], acc[t]);
      }
  };
  int buffer = 0;
  stage(s, columns[0]);
  load_keys(s);
  finish(columns[0]);
  block_sync();
  bool fresh = true;                     // no partial sum left yet
  int first = s.chunk;                   // the first of the block's chunks here
  for (int u = begin;;) {
    const bool last = s.chunk == s.x.chunks - 1;
    if (last || !a.whole) ++u;
    WeightUnit next = s;
    const bool more = u < end && next.next(a, kKeys, kCols);
    const bool other = more && (next.chunk != s.chunk || next.kvh != s.kvh || next.b != s.b);
    if (other) stage(next, columns[buffer ^ 1]);
    const int block = s.block(), key0 = block * kKeys + w * 16 * T;
    const Columns& q = columns[buffer];
    int least = q.least[0];
#pragma unroll
    for (int i = 1; i < W; ++i) least = min(least, q.least[i]);
    if (first_lane(least) >= key0 + 16 * T - 1) {
#pragma unroll
      for (int ct = 0; ct < kCols / 16; ++ct) compute(q, key0, ct, false);
    } else {
      for (int ct = 0; ct < kCols / 16; ++ct)
        if (first_lane(q.most[ct]) >= key0) compute(q, key0, ct, true);
    }
    if (last || !more) {
      const float sum = weight_sums(acc);
#pragma unroll
      for (int t = 0; t < T; ++t) acc[t] = 0.0f;
      const bool whole = last && first == 0;
      const int slot = 2 * blockIdx.x + (fresh ? 0 : 1);
      const int p = key0 + lane;
      if (whole) {
        if (p < s.x.keys && placed) a.weights[((int64_t)s.b * a.kv_heads + s.kvh) * a.row + p] += sum;
      } else {
        a.part[(int64_t)slot * kKeys + w * 16 * T + lane] = placed ? sum : 0.0f;
      }
      if (!a.whole && first == 0 && threadIdx.x == 0)
        a.parts[((int64_t)s.b * a.kv_heads + s.kvh) * a.blocks + block] =
            whole ? u32x2{0, 1}
                  : u32x2{(uint32_t)slot,
                          (uint32_t)(run.owner(u - 1 - s.chunk + s.x.chunks - 1) - blockIdx.x + 1)};
      fresh = false;
      first = 0;
      if (!more) return;
      load_keys(next);
    }
    if (other) {
      buffer ^= 1;
      finish(columns[buffer]);
      block_sync();
    }
    s = next;
  }
}

// The partial sums of the blocks of keys that several workgroups share, added in order.
__global__ __launch_bounds__(weight_keys(kPwManyWaves)) void paged_weight_merge_kernel(PagedWeightArgs a,
                                                                                     int64_t items) {
  constexpr int kKeys = weight_keys(kPwManyWaves);
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int block = (int)(item % a.blocks);
    const int64_t bh = item / a.blocks;
    const int b = (int)(bh / a.kv_heads);
    WeightLengths x;
    x.of(a, kKeys, weight_cols(kPwManyWaves), a.map.starts[b], a.map.counts ? a.map.counts[b] : a.tokens);
    if (block >= x.blocks || x.chunks < 1) continue;
    const u32x2 held = a.parts[item];
    const int slot0 = (int)min(held[0], 2u * a.grid - 1);       // in bounds whatever it holds
    const int parts = min((int)held[1], a.grid - slot0 / 2);
    const int p = block * kKeys + threadIdx.x;
    if (parts <= 1 || p >= x.keys) continue;
    float sum = 0.0f;
    for (int y = 0; y < parts; ++y)
      sum += a.part[(int64_t)(y == 0 ? slot0 : (slot0 & ~1) + 2 * y) * kKeys + threadIdx.x];
    a.weights[bh * a.row + p] += sum;
  }
}

// ------------------------------------------------------------------------- host

struct WeightSizes {
  int64_t chunks, blocks, reach;
  bool few, whole;
  int grid;
};

static bool weight_sizes(const spx_paged_cache& z, int q_heads, WeightSizes& s) {
  if (z.table_width <= 0 || z.page_size <= 0 || z.batch <= 0 || z.tokens <= 0 || q_heads <= 0 ||
      q_heads > 1 << 20 || z.kv_heads <= 0 || q_heads % z.kv_heads != 0)
    return false;
  if ((double)z.batch * z.tokens * q_heads > 0x7fffffff) return false;
  s.reach = (int64_t)z.table_width * z.page_size;
  const int64_t cols = (int64_t)z.tokens * (q_heads / z.kv_heads);
  const bool four = z.key_scales != nullptr;
  s.few = cols <= kPwFewCols;
  s.whole = cols <= kPwWholeCols;
  const int waves = s.whole ? kPwWaves : kPwManyWaves;
  s.chunks = s.few ? 1 : (cols + weight_cols(waves) - 1) / weight_cols(waves);
  const int64_t keys =
      !s.few ? weight_keys(waves) : 16 * (four ? kPwFewTiles<true> : kPwFewTiles<false>);
  s.blocks = (s.reach + keys - 1) / keys;
  // units are counted in 32 bits
  if (s.blocks > 0x7fffffff / s.chunks / ((int64_t)z.batch * z.kv_heads)) return false;
  const int64_t streams = s.blocks * z.batch * z.kv_heads;
  const bool small = z.head_dim == 128;
  const int per_cu = s.few     ? (small ? kPwFewPerSimd<128> : kPwFewPerSimd<256>)
                     : s.whole ? (small ? 3 : 2)
                               : (small ? 2 : 1);
  const int resident = kPwCus * per_cu;
  s.grid = s.few ? (int)std::min<int64_t>((streams + kPwWaves - 1) / kPwWaves, resident)
                 : (int)std::min<int64_t>(s.whole ? streams : streams * s.chunks, resident);
  return true;
}

template <int D, bool kFour>
static int launch_weights(PagedWeightArgs a, const WeightSizes& z, hipStream_t st) {
  if (z.few) {
    a.grid *= kPwWaves;
    a.inv_grid = 1.0 / a.grid;
    paged_weight_few_kernel<D, kFour><<<(unsigned)z.grid, 64 * kPwWaves, 0, st>>>(a);
    return launch_status("paged_accumulate_weights");
  }
  if (a.whole) {
    paged_weight_kernel<D, kFour, kPwWaves><<<(unsigned)a.grid, 64 * kPwWaves, 0, st>>>(a);
  } else {
    paged_weight_kernel<D, kFour, kPwManyWaves><<<(unsigned)a.grid, 64 * kPwManyWaves, 0, st>>>(a);
    const int64_t items = (int64_t)a.batch * a.kv_heads * a.blocks;
    paged_weight_merge_kernel<<<(unsigned)std::min<int64_t>(items, 1 << 20), weight_keys(kPwManyWaves),
                                0, st>>>(a, items);
  }
  return launch_status("paged_accumulate_weights");
}

}  // namespace spx

using namespace spx;

extern "C" int64_t spx_paged_accumulate_weights_workspace_bytes(const spx_paged_cache* cache,
                                                                int q_heads) {
  WeightSizes z;
  if (cache == nullptr || !weight_sizes(*cache, q_heads, z)) return -1;
  if (z.whole) return 0;
  return (int64_t)2 * z.grid * weight_keys(kPwManyWaves) * 4 +
         (int64_t)cache->batch * cache->kv_heads * z.blocks * 8;
}

extern "C" int spx_paged_accumulate_weights(const spx_paged_cache* cache, const void* q,
                                            const int64_t* q_strides, int q_heads, const float* lse,
                                            float scale, void* workspace, float* weights,
                                            int64_t row_stride, void* stream) {
  PagedWeightArgs a{};
  const int status = paged_map(a.map, cache);
  if (status != SPX_OK) return status;
  WeightSizes z;
  SPX_REQUIRE(weight_sizes(*cache, q_heads, z), SPX_EINVAL,
              "bad shape: batch %d tokens %d q_heads %d kv_heads %d", cache->batch, cache->tokens,
              q_heads, cache->kv_heads);
  SPX_REQUIRE(q && q_strides && lse && weights && (workspace || z.whole), SPX_EINVAL,
              "null pointer");
  SPX_REQUIRE((reinterpret_cast<uintptr_t>(q) & 15) == 0 && q_strides[3] == 1 &&
                  ((q_strides[0] | q_strides[1] | q_strides[2]) & 7) == 0,
              SPX_EINVAL,
              "q: base must be 16-byte aligned, the dim stride 1, the others multiples of 8");
  SPX_REQUIRE(((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(weights)) & 3) == 0 &&
                  (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
              SPX_EINVAL, "lse and weights must be 4-byte, the workspace 16-byte aligned");
  SPX_REQUIRE(row_stride >= z.reach, SPX_EINVAL, "weights have %lld slots, the page table reaches %lld",
              (long long)row_stride, (long long)z.reach);
  const bool four = cache->key_scales != nullptr;
  a.q = static_cast<const uint16_t*>(q);
  a.qs_b = q_strides[0]; a.qs_t = q_strides[1]; a.qs_h = q_strides[2];
  a.lse = lse;
  a.key_pages = cache->key_pages; a.value_pages = cache->value_pages;
  a.key_scales = static_cast<const uint8_t*>(cache->key_scales);
  a.value_scales = static_cast<const uint8_t*>(cache->value_scales);
  a.batch = cache->batch; a.tokens = cache->tokens;
  a.q_heads = q_heads; a.kv_heads = cache->kv_heads; a.group = q_heads / cache->kv_heads;
  a.whole = z.whole;
  a.blocks = (int)z.blocks;
  a.grid = z.grid;
  a.inv_grid = 1.0 / a.grid;
  a.inv_group = 1.0 / a.group;
  const double scale_log2 = (double)scale * 1.4426950408889634;
  a.scale = (float)scale_log2;
  a.scale_rest = a.scale == 0.0f ? 0.0f : (float)((scale_log2 - (double)a.scale) / (double)a.scale);
  a.weights = weights;
  a.row = row_stride;
  a.part = static_cast<float*>(workspace);
  a.parts = reinterpret_cast<u32x2*>(a.part + (int64_t)2 * a.grid * weight_keys(kPwManyWaves));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (cache->head_dim == 128)
    return four ? launch_weights<128, true>(a, z, st) : launch_weights<128, false>(a, z, st);
  return four ? launch_weights<256, true>(a, z, st) : launch_weights<256, false>(a, z, st);
}
