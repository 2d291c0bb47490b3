// Eviction from the paged cache: which tokens of a KV head stay, and where they go.
//
// Of the `length` tokens of a sequence each KV head keeps `budget`: those whose position is below
// `sinks` or among the last `recent`, then those of the largest weight, the lower slot first among
// equals. Slots below the budget that become free are filled with the tokens kept behind it, the j-th
// with the j-th: no row is read that another move writes, and nothing else moves.
//
// One workgroup per (sequence, KV head) finds the budget-th largest rank of its weights: histograms of
// eight bits until at most 64 tokens are left to choose from, which one wave ranks. It then counts and
// writes the list of moves, in the order of the slots, and clears the ledger of the tokens behind the
// budget that it drops. The kept ones move in a launch of their own, row and ledger, so that both
// may be in place.
//
// Bound by the walks' instructions and serial steps: a row is one workgroup's, so few long rows leave
// most CUs idle (1 x 4 heads of 32640 tokens to 4096: 30.4 us, 16 waves, + 5.6 for the moves; 64 x 8
// heads of 2112 to 2048: 16.3 + 8.4, the bytes of both 8). Rows shared by workgroups (one histogram of
// more bits over all of them, few candidates left) would take a launch or two more; not built, and not
// measured.
#include <algorithm>

#include "paged_moves.h"
#include "paged_tiles.h"

namespace spx {

constexpr int kBins = 256;
constexpr int kFew = 64;                 // tokens that one wave ranks

struct EvictArgs {
  PagedMap map;
  int64_t row;                           // elements of a row of weights and positions
  int budget, recent, sinks, room;
  const float* weights;                  // [B, Hkv, row]
  const int32_t* positions;              // the same, or null
  const int32_t* seen;                   // [B], or null: the lengths
  float* weights_out;
  int32_t* positions_out;
  int32_t* lengths_out;                  // [B]
  int32_t* counts;                       // [B, Hkv]
  u32x2* moves;                          // [B, Hkv, room]
};

struct EvictRow {
  const float* weights;
  const int32_t* positions;
  int length, seen, sinks, since;        // since: the first of the recent positions

  __device__ __forceinline__ int told(int slot) const { return positions ? positions[slot] : -1; }
  __device__ __forceinline__ int position(int slot) const {
    const int x = told(slot);
    return x >= 0 ? x : seen - length + slot;
  }
  // Ranks as unsigned numbers: NaN last, -0 as 0, protected ones first.
  __device__ __forceinline__ uint32_t rank(float weight, int p) const {
    const float w = weight + 0.0f;
    const uint32_t u = __float_as_uint(w);
    const uint32_t ordered = w != w ? 0 : u >> 31 ? ~u : u | 0x80000000u;
    return p < sinks || p >= since ? 0xffffffffu : ordered;
  }
  __device__ __forceinline__ uint32_t rank(int slot) const {
    return rank(weights[slot], position(slot));
  }
};

// W waves. Rows of up to kSlots tokens have their ranks in LDS, longer ones form them anew from memory
// in each walk. A bin has kCopies, in banks of their own: few lanes of one digit meet.
// (Ranks in registers: 32640 tokens 53 us, the walks unrolled 64 times and fetched once.)
template <int W, int kSlots, int kCopies>
__global__ __launch_bounds__(64 * W) void paged_evict_kernel(EvictArgs a) {
  constexpr int kThreads = 64 * W, kChunk = 4 * kWave;          // slots of a wave's step, 4 a lane
  __shared__ __align__(16) uint32_t ranks[kSlots];
  __shared__ __align__(16) uint32_t bins[kBins * kCopies];
  __shared__ int sums[kBins];
  __shared__ int found[3];               // digit, how many of it stay, how many there are
  __shared__ uint32_t few[kFew];
  __shared__ int few_slot[kFew];
  __shared__ int few_count;
  __shared__ int wave_equal[2][W], wave_above[2][W];            // below the budget, behind it
  __shared__ int lost;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t bh = blockIdx.x;
  const int b = (int)(bh / a.map.kv_heads), head = (int)(bh % a.map.kv_heads);
  const int length = a.map.starts[b];
  EvictRow row;
  row.weights = a.weights + bh * a.row;
  row.positions = a.positions ? a.positions + bh * a.row : nullptr;
  row.length = length;
  row.seen = a.seen ? a.seen[b] : length;
  row.sinks = a.sinks;
  row.since = row.seen - a.recent;
  float* weights_out = a.weights_out + bh * a.row;
  int32_t* positions_out = a.positions_out + bh * a.row;
  if (tid == 0) lost = few_count = 0;
  block_sync();
  bool cut = length > a.budget && length <= a.map.capacity();
  if (cut) {                             // a sequence with a token that has no place is left alone
    const int pages = ((length - 1) >> a.map.page_shift) + 1;
    bool bad = false;
    for (int i = tid; i < pages; i += kThreads) bad |= a.map.page(b, i << a.map.page_shift) < 0;
    if (bad) lost = 1;
    block_sync();
    cut = lost == 0;
  }
  if (tid == 0 && head == 0) a.lengths_out[b] = cut ? a.budget : length;
  if (!cut) {
    if (tid == 0) a.counts[bh] = 0;
    const int left = (int)min((int64_t)max(length, 0), a.row);
    for (int i = tid; i < left; i += kThreads) {
      const float x = row.weights[i];
      const int p = row.told(i);
      weights_out[i] = x;
      positions_out[i] = p;
    }
    return;
  }
  const bool held = length <= kSlots;
  // A wave has a run of slots, a lane four of every 256. Slots behind the length count as rank 0, the
  // least, and come after all tokens: as the budget is below the length none of them is chosen.
  const int part = ((length + W - 1) / W + kChunk - 1) / kChunk * kChunk;
  const int begin = w * part, end = begin < length ? begin + part : begin;
  for (int i = tid; i < kBins * kCopies / 4; i += kThreads) reinterpret_cast<u32x4*>(bins)[i] = u32x4{};
  block_sync();
  // Ranks into LDS and their first digits counted; slots below the budget keep what they have for
  // now. Loads first, kAtOnce at a time: the stores between them may be to the same tensors.
  constexpr int kAtOnce = 16;
  for (int i0 = tid; i0 < W * part; i0 += kAtOnce * kThreads) {
    float x[kAtOnce];
    int told[kAtOnce];
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      const int i = min(i0 + n * kThreads, length - 1);
      x[n] = row.weights[i];
      told[n] = row.told(i);
    }
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      const int i = i0 + n * kThreads;
      const int p = told[n] >= 0 ? told[n] : row.seen - length + i;
      const uint32_t r = i < length ? row.rank(x[n], p) : 0;
      if (held && i < kSlots) ranks[i] = r;
      if (i < W * part) atomicAdd(&bins[(r >> 24) * kCopies + lane % kCopies], 1u);
      if (i < a.budget) {
        weights_out[i] = x[n];
        positions_out[i] = p;
      }
    }
  }
  const auto four = [&](int i, uint32_t (&r)[4]) {
    if (held) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(ranks + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = x[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = i + e < length ? row.rank(i + e) : 0;
    }
  };
  // `need` tokens of the ranks that begin with the bits `prefix` above `shift` stay
  uint32_t prefix = 0;
  int need = a.budget;
  int equal[2] = {0, 0}, over[2] = {0, 0};           // the lane's: below the budget, behind it
  bool counted = false;
  for (int shift = 24;; shift -= 8) {
    block_sync();
    {                                    // W / 4 lanes a bin
      constexpr int kLanes = W / 4;
      const int bin = tid / kLanes;
      int sum = 0;
#pragma unroll
      for (int i = 0; i < kCopies / kLanes; ++i)
        sum += (int)bins[bin * kCopies + (kLanes * (i + bin) + tid % kLanes) % kCopies];
#pragma unroll
      for (int o = 1; o < kLanes; o *= 2) sum += __shfl_xor(sum, o);
      if (tid % kLanes == 0) sums[bin] = sum;
    }
    block_sync();
    if (w == 0) {                        // lane i: digits 255 - 4 i .. 252 - 4 i
      int x[4], all = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) all += x[e] = sums[255 - 4 * lane - e];
      int before = wave_prefix(all) - all;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (before < need && need <= before + x[e]) {
          found[0] = 255 - 4 * lane - e;
          found[1] = need - before;
          found[2] = x[e];
        }
        before += x[e];
      }
    } else {
      for (int i = tid - kWave; i < kBins * kCopies / 4; i += kThreads - kWave)
        reinterpret_cast<u32x4*>(bins)[i] = u32x4{};
    }
    block_sync();
    prefix |= (uint32_t)found[0] << shift;
    need = found[1];
    const int count = found[2];
    if (shift == 0) break;
    const uint32_t digits = 0xffffffffu << shift;
    if (count <= kFew) {                 // one wave ranks what is left, each against all
      for (int i0 = begin; i0 < end; i0 += kChunk) {
        const int i = i0 + 4 * lane;
        const bool below = i0 + kChunk <= a.budget;
        uint32_t r[4];
        four(i, r);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int more = r[e] > (prefix | ~digits);
          const bool low = below || i + e < a.budget;
          over[0] += low ? more : 0;
          over[1] += low ? 0 : more;
          if ((r[e] & digits) == prefix) {
            const int at = atomicAdd(&few_count, 1);
            few[at] = r[e];
            few_slot[at] = i + e;
          }
        }
      }
      block_sync();
      if (w == 0) {
        const uint32_t mine = lane < count ? few[lane] : 0;
        int larger = 0, same = 0;
        for (int i = 0; i < count; ++i) {
          const uint32_t x = few[i];
          larger += x > mine;
          same += x == mine;
        }
        if (lane < count && larger < need && need <= larger + same) {
          found[0] = (int)mine;
          found[1] = need - larger;
        }
      }
      block_sync();
      prefix = (uint32_t)found[0];
      need = found[1];
      for (int i = 0; i < count; ++i) {  // those of the wave's run, counted by its first lane
        const int slot = few_slot[i];
        const bool low = slot < a.budget;
        if (lane != 0 || slot < begin || slot >= end) continue;
        if (few[i] == prefix) ++equal[low ? 0 : 1];
        if (few[i] > prefix) ++over[low ? 0 : 1];
      }
      counted = true;
      break;
    }
#pragma unroll 2
    for (int i0 = begin; i0 < end; i0 += kChunk) {
      const int i = i0 + 4 * lane;
      uint32_t r[4];
      four(i, r);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((r[e] & digits) == prefix)
          atomicAdd(&bins[(r[e] >> (shift - 8) & 255) * kCopies + lane % kCopies], 1u);
    }
  }
  // `need` of the tokens of rank `prefix` stay, the lowest slots
  if (!counted) {
    for (int i0 = begin; i0 < end; i0 += kChunk) {
      const int i = i0 + 4 * lane;
      uint32_t r[4];
      four(i, r);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool low = i + e < a.budget;
        const int same = r[e] == prefix, more = r[e] > prefix;
        equal[0] += low ? same : 0;
        equal[1] += low ? 0 : same;
        over[0] += low ? more : 0;
        over[1] += low ? 0 : more;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int x = wave_prefix(equal[e]), y = wave_prefix(over[e]);
    if (lane == kWave - 1) {
      wave_equal[e][w] = x;
      wave_above[e][w] = y;
    }
  }
  block_sync();
  // equal ones, free slots and moves before this wave's run; all moves
  int equals = 0, to = 0, from = 0, moves = 0, same_before = 0, kept_low = 0;
  for (int x = 0; x < W; ++x) {
    if (x == w) {
      equals = same_before;
      to = min(begin, a.budget) - kept_low;
      from = moves;
    }
    const int all = wave_equal[0][x] + wave_equal[1][x];
    const int keep = min(max(need - same_before, 0), all), low = min(keep, wave_equal[0][x]);
    kept_low += wave_above[0][x] + low;
    moves += wave_above[1][x] + keep - low;
    same_before += all;
  }
  if (tid == 0) a.counts[bh] = moves;
  u32x2* list = a.moves + bh * a.room;
  const bool wide =
      ((reinterpret_cast<uintptr_t>(weights_out) | reinterpret_cast<uintptr_t>(positions_out)) & 15) == 0;
  for (int i0 = begin; i0 < end; i0 += kChunk) {
    const int i = i0 + 4 * lane;
    uint32_t r[4];
    four(i, r);
    int mine = 0, before = 0;            // equal ones: the lane's, those of the lanes before it
#pragma unroll
    for (int e = 0; e < 4; ++e) mine += r[e] == prefix;
    if (__any(mine != 0)) {
      const int up_to = wave_prefix(mine);
      before = equals + up_to - mine;
      equals += __builtin_amdgcn_readlane(up_to, kWave - 1);
    }
    bool hole[4], far[4], gone[4];
    int both = 0;                        // holes, and kept ones behind the budget << 16
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool low = i + e < a.budget, same = r[e] == prefix;
      const bool kept = r[e] > prefix || (same && before < need);
      before += same;
      hole[e] = !kept && low;
      far[e] = kept && !low;
      both += (int)hole[e] + ((int)far[e] << 16);
      gone[e] = !kept && !low && i + e < length;     // dropped; what is kept there, moves
    }
    if (wide && gone[0] && gone[1] && gone[2] && gone[3]) {
      *reinterpret_cast<u32x4*>(weights_out + i) = u32x4{};
      *reinterpret_cast<u32x4*>(positions_out + i) = ~u32x4{};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (gone[e]) {
          weights_out[i + e] = 0.0f;
          positions_out[i + e] = -1;
        }
    }
    if (!__any(both != 0)) continue;
    const int up_to = wave_prefix(both);
    int h = to + ((up_to - both) & 0xffff), f = from + ((up_to - both) >> 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (hole[e]) reinterpret_cast<uint32_t*>(list + h)[0] = (uint32_t)(i + e);
      if (far[e]) reinterpret_cast<uint32_t*>(list + f)[1] = (uint32_t)(i + e);
      h += hole[e];
      f += far[e];
    }
    const int last = __builtin_amdgcn_readlane(up_to, kWave - 1);
    to += last & 0xffff;
    from += last >> 16;
  }
}

static int64_t evict_room(const spx_paged_cache& z, int budget) {
  const int64_t reach = (int64_t)z.table_width * z.page_size;
  return std::max<int64_t>(1, std::min<int64_t>(budget, reach - budget));
}

}  // namespace spx

using namespace spx;

extern "C" int64_t spx_paged_evict_workspace_bytes(const spx_paged_cache* cache, int budget) {
  if (cache == nullptr || cache->table_width <= 0 || cache->page_size <= 0 || cache->batch <= 0 ||
      cache->kv_heads <= 0 || budget <= 0)
    return -1;
  const int64_t rows = (int64_t)cache->batch * cache->kv_heads;
  return rows * 8 + rows * evict_room(*cache, budget) * 8;
}

extern "C" int spx_paged_evict(const spx_paged_cache* cache, const float* weights,
                               const int32_t* positions, int64_t row_stride, const int32_t* seen,
                               int budget, int recent, int sinks, void* workspace, float* weights_out,
                               int32_t* positions_out, int32_t* lengths_out, void* stream) {
  EvictArgs a{};
  const int status = paged_map(a.map, cache);
  if (status != SPX_OK) return status;
  SPX_REQUIRE(weights && weights_out && positions_out && lengths_out && workspace, SPX_EINVAL,
              "null pointer");
  SPX_REQUIRE(((reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(positions) |
                reinterpret_cast<uintptr_t>(seen) | reinterpret_cast<uintptr_t>(weights_out) |
                reinterpret_cast<uintptr_t>(positions_out) | reinterpret_cast<uintptr_t>(lengths_out)) &
               3) == 0 && (reinterpret_cast<uintptr_t>(workspace) & 7) == 0,
              SPX_EINVAL, "tensors must be 4-byte, the workspace 8-byte aligned");
  SPX_REQUIRE(row_stride >= (int64_t)cache->table_width * cache->page_size, SPX_EINVAL,
              "weights have %lld slots, the page table reaches %lld", (long long)row_stride,
              (long long)cache->table_width * cache->page_size);
  SPX_REQUIRE(budget > 0 && recent >= 0 && sinks >= 0 && (int64_t)recent + sinks <= budget, SPX_EINVAL,
              "budget %d must be positive and hold the %d recent and %d first tokens", budget, recent,
              sinks);
  const int64_t rows = (int64_t)cache->batch * cache->kv_heads;
  SPX_REQUIRE(rows <= 1 << 21, SPX_EINVAL, "%lld sequences x heads are more than 2^21",
              (long long)rows);
  a.row = row_stride;
  a.budget = budget; a.recent = recent; a.sinks = sinks;
  a.room = (int)evict_room(*cache, budget);
  a.weights = weights; a.positions = positions; a.seen = seen;
  a.weights_out = weights_out; a.positions_out = positions_out; a.lengths_out = lengths_out;
  a.counts = static_cast<int32_t*>(workspace);
  a.moves = reinterpret_cast<u32x2*>(static_cast<uint8_t*>(workspace) + rows * 8);
  hipStream_t st = static_cast<hipStream_t>(stream);
  // Up to 4096 tokens four waves a row, several rows on a compute unit; 128 KB of LDS hold 32768.
  if ((int64_t)cache->table_width * cache->page_size <= 4096)
    paged_evict_kernel<4, 4096, 8><<<(unsigned)rows, 256, 0, st>>>(a);
  else
    paged_evict_kernel<16, 32768, 16><<<(unsigned)rows, 1024, 0, st>>>(a);
  const int launched = launch_status("paged_evict");
  if (launched != SPX_OK) return launched;
  MoveArgs m{};
  m.map = a.map;
  m.batch = cache->batch;
  m.room = a.room;
  m.pages = PagePointers{cache->key_pages, cache->value_pages, cache->key_scales, cache->value_scales};
  m.counts = a.counts;
  m.moves = a.moves;
  m.row = a.row;
  m.seen = seen;
  m.weights = weights;
  m.positions = positions;
  m.weights_out = weights_out;
  m.positions_out = positions_out;
  return launch_moves(m, cache->head_dim, st);
}
