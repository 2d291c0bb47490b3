// Attention weight that cached tokens gather: with the LSE of an attention call over the paged cache,
//
//   weights[b, kvh, p] += sum over rows (i, h of the group) that see p of exp(scale q k_p - lse).
//
// Columns n = i group + h of a KV head, 16 to a matrix tile; a wave holds 32 keys and walks the
// columns. v_mfma_f32_16x16x32_bf16 with Q as A and K as B operand: the scores of a key lie in one
// lane's four registers, so the sum over columns is in the lane but for the lane groups at the end.
// Q comes from LDS, 128 columns at a time, K straight from the pages into registers.
//
// Work: a stream is a (sequence, KV head, 128 or 256 keys), its units chunks of 128 columns. The units
// of all streams are dealt in equal runs to one grid; where a stream has one unit (decode steps) every
// workgroup adds to the weights itself, else streams that cross workgroups leave at most two partial
// sums per workgroup, added in order by a second kernel.
#include <algorithm>
#include <cmath>

#include "paged_tiles.h"

namespace spx {

constexpr int kPwCols = 128;             // columns of a unit
constexpr int kPwCus = 256;
constexpr int kPwTiles = 2;              // of 16 keys, a wave's

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
  int cols, chunks;                      // tokens x group, chunks of them at most
  int blocks;                            // blocks of keys that the table reaches
  int grid;
  double inv_grid, inv_group;
  float scale, scale_low;                // scale log2(e) in two parts
  float* weights;                        // [B, Hkv, row]
  int64_t row;
  float* part;                           // [2 grid][keys of a block]
  u32x2* parts;                          // [B, Hkv, blocks]
};

struct WeightLengths {
  int start, live, keys, blocks, chunks;
  __device__ __forceinline__ void of(const PagedWeightArgs& a, int block, int start_, int count) {
    start = start_;
    const int64_t room = a.map.capacity() - start;
    live = start < 0 ? 0
                     : max(0, min(min(count, a.tokens), (int)min(room, (int64_t)a.tokens)));
    keys = live > 0 ? start + live : 0;
    blocks = (keys + block - 1) / block;
    chunks = (live * a.group + kPwCols - 1) / kPwCols;
  }
  __device__ __forceinline__ void load(const PagedWeightArgs& a, int block, int b) {
    of(a, block, scalar_load(a.map.starts + b),
       a.map.counts ? scalar_load(a.map.counts + b) : a.tokens);
  }
};

struct WeightScan {                      // the units of 64 sequences, one a lane
  int units, sum;
  __device__ __forceinline__ void load(const PagedWeightArgs& a, int block, int b) {
    WeightLengths x;
    int start = -1, count = a.tokens;
    if (b < a.batch) {
      start = a.map.starts[b];
      if (a.map.counts) count = a.map.counts[b];
    }
    x.of(a, block, start, count);
    units = x.blocks * x.chunks * a.kv_heads;
    sum = wave_prefix(units);
  }
  __device__ __forceinline__ int total() const { return __builtin_amdgcn_readlane(sum, kWave - 1); }
};

struct WeightUnit {
  WeightLengths x;
  int b, kvh, at, chunk;                 // at: which of the blocks, in the order of the runs

  __device__ __forceinline__ bool find(const PagedWeightArgs& a, int block, int lane, WeightScan scan,
                                       int u) {
    int before = 0, b0 = 0;
    uint64_t past;
    while (!(past = __ballot(before + scan.sum > u))) {
      before += scan.total();
      b0 += kWave;
      if (b0 >= a.batch) return false;
      scan.load(a, block, b0 + lane);
    }
    const int l = __builtin_ctzll(past);
    b = b0 + l;
    before += __builtin_amdgcn_readlane(scan.sum - scan.units, l);
    x.load(a, block, b);
    if (x.blocks <= 0 || x.chunks <= 0 || u < before) return false;
    const int stream = (u - before) / x.chunks;
    chunk = u - before - stream * x.chunks;
    kvh = stream / x.blocks;
    at = stream - kvh * x.blocks;
    return kvh < a.kv_heads;
  }
  __device__ __forceinline__ bool next(const PagedWeightArgs& a, int block) {
    if (++chunk < x.chunks) return true;
    chunk = 0;
    if (++at < x.blocks) return true;
    at = 0;
    if (++kvh < a.kv_heads) return true;
    kvh = 0;
    do {
      if (++b >= a.batch) return false;
      x.load(a, block, b);
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

template <int D, bool kFour, int W>
__global__ __launch_bounds__(64 * W) void paged_weight_kernel(PagedWeightArgs a) {
  constexpr int kBlockKeys = 16 * kPwTiles * W, KK = D / 32, kRowChunks = D / 8;
  __shared__ __align__(16) uint16_t qs[kPwCols * D];
  __shared__ __align__(16) float lse_hi[kPwCols], lse_lo[kPwCols];
  __shared__ __align__(16) int last_key[kPwCols];               // that a column sees; -1: none
  const int tid = threadIdx.x, lane = tid & 63, w = first_lane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  WeightScan scan;
  scan.load(a, kBlockKeys, lane);
  int total = scan.total();
  for (int b0 = kWave; b0 < a.batch; b0 += kWave) {
    WeightScan more;
    more.load(a, kBlockKeys, b0 + lane);
    total += more.total();
  }
  const WeightRun run(total, a.grid, a.inv_grid);
  const int begin = run.begin(blockIdx.x), end = run.begin(blockIdx.x + 1);
  WeightUnit s;
  if (begin >= end || !s.find(a, kBlockKeys, lane, scan, begin)) return;
  int held_b = -1, held_kvh = 0, held_chunk = 0;                // whose columns are in LDS
  KeyTile<D, kFour> key[kPwTiles];
  bool placed[kPwTiles];
  const auto load_keys = [&](const WeightUnit& s) {
    const HeadPages<D, kFour> pages(a, s.kvh);
    const int key0 = s.block() * kBlockKeys + w * 16 * kPwTiles;
#pragma unroll
    for (int t = 0; t < kPwTiles; ++t) {
      const int p = key0 + 16 * t;
      const int id = a.map.uniform_page(s.b, min(p, s.x.keys - 1));
      placed[t] = id >= 0;
      key[t].load(pages, pages.row(max(id, 0), p), c, g);
    }
  };
  load_keys(s);
  float acc[kPwTiles] = {};
  bool fresh = true;                     // acc holds nothing of the stream
  int first = s.chunk;                   // the first of its chunks here
  for (int u = begin;;) {
    const int block = s.block(), key0 = block * kBlockKeys + w * 16 * kPwTiles;
    if (s.b != held_b || s.kvh != held_kvh || s.chunk != held_chunk) {
      block_sync();                      // the last columns have been read
      held_b = s.b;
      held_kvh = s.kvh;
      held_chunk = s.chunk;
      const int n0 = s.chunk * kPwCols;
      const int rows = min((s.x.live * a.group - n0 + 15) & ~15, kPwCols);
      for (int i = tid; i < rows * kRowChunks; i += 64 * W) {
        const int n = n0 + i / kRowChunks, piece = i % kRowChunks;
        const int token = divide(n, a.group, a.inv_group);
        const int head = s.kvh * a.group + n - token * a.group;
        u32x4 x{};
        if (token < s.x.live)
          x = *reinterpret_cast<const u32x4*>(a.q + s.b * a.qs_b + token * a.qs_t + head * a.qs_h +
                                              8 * piece);
        *reinterpret_cast<u32x4*>(qs + (n - n0) * D + ((piece ^ (n & 15)) << 3)) = x;
      }
      for (int i = tid; i < rows; i += 64 * W) {
        const int n = n0 + i, token = divide(n, a.group, a.inv_group);
        float lse = -INFINITY;
        if (token < s.x.live)
          lse = a.lse[((int64_t)s.b * a.tokens + token) * a.q_heads + s.kvh * a.group + n -
                      token * a.group];
        const float hi = lse * kLog2e;
        // log2(e) is kLog2e + 1.925963033500e-8
        const float lo = __builtin_fmaf(lse, kLog2e, -hi) + lse * 1.925963033500e-8f;
        lse_hi[i] = hi;
        lse_lo[i] = __builtin_isinf(hi) ? 0.0f : lo;
        last_key[i] = lse == -INFINITY ? -1 : s.x.start + token;
      }
      block_sync();
    }
    const int n0 = s.chunk * kPwCols, columns = min(s.x.live * a.group - n0, kPwCols);
    for (int ct = 0; ct < columns; ct += 16) {
      const int last_token = divide(n0 + min(ct + 16, columns) - 1, a.group, a.inv_group);
      if (key0 > s.x.start + last_token) continue;
      f32x4 x[kPwTiles];
#pragma unroll
      for (int t = 0; t < kPwTiles; ++t) x[t] = f32x4{};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const int piece = KeyTile<D, kFour>::dim(kk, g) / 8;
        const u32x4 q = *reinterpret_cast<const u32x4*>(qs + (ct + c) * D + ((piece ^ c) << 3));
#pragma unroll
        for (int t = 0; t < kPwTiles; ++t) x[t] = mfma16(q, key[t].operand(kk, g), x[t]);
      }
      const f32x4 hi = *reinterpret_cast<const f32x4*>(lse_hi + ct + 4 * g);
      const f32x4 lo = *reinterpret_cast<const f32x4*>(lse_lo + ct + 4 * g);
      typedef int i32x4 __attribute__((ext_vector_type(4)));
      const i32x4 see = *reinterpret_cast<const i32x4*>(last_key + ct + 4 * g);
#pragma unroll
      for (int t = 0; t < kPwTiles; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float y = __builtin_fmaf(x[t][r], a.scale, -hi[r]) +
                          __builtin_fmaf(x[t][r], a.scale_low, -lo[r]);
          const float p = exp2_fast(y);
          acc[t] += key0 + 16 * t + c <= see[r] ? p : 0.0f;
        }
    }
    const bool last = s.chunk == s.x.chunks - 1;
    ++u;
    if (last || u >= end) {
      float sum[kPwTiles];
#pragma unroll
      for (int t = 0; t < kPwTiles; ++t) {
        sum[t] = acc[t] + __shfl_xor(acc[t], 16);
        sum[t] += __shfl_xor(sum[t], 32);
        acc[t] = 0.0f;
      }
      const bool whole = last && first == 0;
      const int slot = 2 * blockIdx.x + (fresh ? 0 : 1);
      const int p = key0 + 16 * g + c;
      const float mine = g == 0 ? sum[0] : sum[1];
      if (g < kPwTiles) {
        if (whole) {
          if (p < s.x.keys && (g == 0 ? placed[0] : placed[1]))
            a.weights[((int64_t)s.b * a.kv_heads + s.kvh) * a.row + p] += mine;
        } else {
          a.part[(int64_t)slot * kBlockKeys + w * 16 * kPwTiles + 16 * g + c] =
              (g == 0 ? placed[0] : placed[1]) ? mine : 0.0f;
        }
      }
      if (!whole && first == 0 && tid == 0)
        a.parts[((int64_t)s.b * a.kv_heads + s.kvh) * a.blocks + block] =
            u32x2{(uint32_t)slot, (uint32_t)(run.owner(u - 1 - s.chunk + s.x.chunks - 1) - blockIdx.x + 1)};
      else if (whole && a.chunks > 1 && tid == 0)
        a.parts[((int64_t)s.b * a.kv_heads + s.kvh) * a.blocks + block] = u32x2{0, 1};
      fresh = false;
      first = 0;
      if (u >= end || !s.next(a, kBlockKeys)) return;
      load_keys(s);
    } else if (!s.next(a, kBlockKeys)) {
      return;
    }
  }
}

// The partial sums of the blocks of keys that several workgroups share, added in order.
template <int W>
__global__ __launch_bounds__(16 * kPwTiles * W) void paged_weight_merge_kernel(PagedWeightArgs a,
                                                                              int64_t items) {
  constexpr int kBlockKeys = 16 * kPwTiles * W;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int block = (int)(item % a.blocks);
    const int64_t bh = item / a.blocks;
    const int b = (int)(bh / a.kv_heads);
    WeightLengths x;
    x.of(a, kBlockKeys, a.map.starts[b], a.map.counts ? a.map.counts[b] : a.tokens);
    if (block >= x.blocks || x.chunks <= 1) continue;
    const u32x2 held = a.parts[item];
    const int slot0 = (int)min(held[0], 2u * a.grid - 1);       // in bounds whatever it holds
    const int parts = min((int)held[1], a.grid - slot0 / 2);
    const int p = block * kBlockKeys + threadIdx.x;
    if (parts <= 1 || p >= x.keys) continue;
    float sum = 0.0f;
    for (int y = 0; y < parts; ++y)
      sum += a.part[(int64_t)(y == 0 ? slot0 : (slot0 & ~1) + 2 * y) * kBlockKeys + threadIdx.x];
    a.weights[bh * a.row + p] += sum;
  }
}

// ------------------------------------------------------------------------- host

constexpr int kPwFew = 4, kPwMany = 8;   // waves of a workgroup

struct WeightSizes {
  int64_t reach, chunks, blocks, units;
  int waves, grid;
};

static bool weight_sizes(const spx_paged_cache& z, int q_heads, WeightSizes& s) {
  if (z.table_width <= 0 || z.page_size <= 0 || z.batch <= 0 || z.tokens <= 0 || q_heads <= 0 ||
      q_heads > 1 << 20 || z.kv_heads <= 0 || q_heads % z.kv_heads != 0)
    return false;
  if ((double)z.batch * z.tokens * q_heads > 0x7fffffff) return false;
  s.reach = (int64_t)z.table_width * z.page_size;
  const int64_t cols = (int64_t)z.tokens * (q_heads / z.kv_heads);
  s.chunks = (cols + kPwCols - 1) / kPwCols;
  s.waves = s.chunks > 1 ? kPwMany : kPwFew;
  const int64_t keys = 16 * kPwTiles * s.waves;
  s.blocks = (s.reach + keys - 1) / keys;
  // units are counted in 32 bits
  if (s.blocks > 0x7fffffff / s.chunks / ((int64_t)z.batch * z.kv_heads)) return false;
  s.units = s.blocks * s.chunks * z.batch * z.kv_heads;
  s.grid = (int)std::min<int64_t>(s.units, kPwCus * (s.waves == kPwFew ? 4 : 2));
  return true;
}

template <int D, bool kFour, int W>
static int launch_weights(const PagedWeightArgs& a, hipStream_t st) {
  paged_weight_kernel<D, kFour, W><<<(unsigned)a.grid, 64 * W, 0, st>>>(a);
  if (a.chunks > 1) {
    const int64_t items = (int64_t)a.batch * a.kv_heads * a.blocks;
    paged_weight_merge_kernel<W>
        <<<(unsigned)std::min<int64_t>(items, 1 << 20), 16 * kPwTiles * W, 0, st>>>(a, items);
  }
  return launch_status("paged_accumulate_weights");
}

template <int D, bool kFour>
static int launch_weights(const PagedWeightArgs& a, int waves, hipStream_t st) {
  return waves == kPwFew ? launch_weights<D, kFour, kPwFew>(a, st)
                         : launch_weights<D, kFour, kPwMany>(a, st);
}

}  // namespace spx

using namespace spx;

extern "C" int64_t spx_paged_accumulate_weights_workspace_bytes(const spx_paged_cache* cache,
                                                                int q_heads) {
  WeightSizes z;
  if (cache == nullptr || !weight_sizes(*cache, q_heads, z)) return -1;
  if (z.chunks == 1) return 0;
  return ((int64_t)2 * z.grid * 16 * kPwTiles * z.waves) * 4 +
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
  SPX_REQUIRE(q && q_strides && lse && weights && (workspace || z.chunks == 1), SPX_EINVAL,
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
  a.cols = cache->tokens * a.group;
  a.chunks = (int)z.chunks;
  a.blocks = (int)z.blocks;
  a.grid = z.grid;
  a.inv_grid = 1.0 / a.grid;
  a.inv_group = 1.0 / a.group;
  const double scale_log2 = (double)scale * 1.4426950408889634;
  a.scale = (float)scale_log2;
  a.scale_low = (float)(scale_log2 - (double)a.scale);
  a.weights = weights;
  a.row = row_stride;
  a.part = static_cast<float*>(workspace);
  a.parts = reinterpret_cast<u32x2*>(a.part + (int64_t)2 * a.grid * 16 * kPwTiles * z.waves);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (cache->head_dim == 128)
    return four ? launch_weights<128, true>(a, z.waves, st) : launch_weights<128, false>(a, z.waves, st);
  return four ? launch_weights<256, true>(a, z.waves, st) : launch_weights<256, false>(a, z.waves, st);
}
