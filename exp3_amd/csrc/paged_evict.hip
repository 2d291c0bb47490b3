// Eviction from the paged cache: which tokens of a KV head stay, and where they go.
//
// Of the `length` tokens of a sequence each KV head keeps `budget`: those whose position is below
// `sinks` or among the last `recent`, then those of the largest weight, the lower slot first among
// equals. Slots below the budget that become free are filled with the tokens kept behind it, the j-th
// with the j-th: no row is read that another move writes, and nothing else moves.
//
// One workgroup per (sequence, KV head) finds the budget-th largest rank of its weights digit by digit
// (histograms of eight bits), then walks the slots once to count and once to write the list of moves;
// the rows themselves move in a launch of their own.
#include <algorithm>

#include "paged_moves.h"

namespace spx {

constexpr int kEvictThreads = 1024, kEvictWaves = kEvictThreads / kWave;
constexpr int kBins = 256, kCopies = 32;

struct EvictArgs {
  PagedMap map;
  int64_t row;                           // elements of a row of weights and positions
  int batch, budget, recent, sinks, room;
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
  __device__ __forceinline__ uint32_t rank(int slot) const {
    const int p = position(slot);
    const float w = weights[slot] + 0.0f;
    const uint32_t u = __float_as_uint(w);
    const uint32_t ordered = w != w ? 0 : u >> 31 ? ~u : u | 0x80000000u;
    return p < sinks || p >= since ? 0xffffffffu : ordered;
  }
};

__global__ __launch_bounds__(kEvictThreads) void paged_evict_kernel(EvictArgs a) {
  __shared__ uint32_t bins[kBins][kCopies];
  __shared__ int sums[kBins];
  __shared__ int found[2];               // digit, and how many of it stay
  __shared__ int wave_equal[2][kEvictWaves], wave_above[2][kEvictWaves];   // below the budget, behind it
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
  if (tid == 0) lost = 0;
  block_sync();
  bool cut = length > a.budget && length <= a.map.capacity();
  if (cut) {                             // a sequence with a token that has no place is left alone
    const int pages = ((length - 1) >> a.map.page_shift) + 1;
    bool bad = false;
    for (int i = tid; i < pages; i += kEvictThreads) bad |= a.map.page(b, i << a.map.page_shift) < 0;
    if (bad) lost = 1;
    block_sync();
    cut = lost == 0;
  }
  const int left = cut ? a.budget : length;
  if (tid == 0 && head == 0) a.lengths_out[b] = left;
  if (!cut) {
    if (tid == 0) a.counts[bh] = 0;
    for (int64_t i = tid; i < a.row; i += kEvictThreads) {
      const bool here = i < left;
      const float x = here ? row.weights[i] : 0.0f;
      const int p = here ? row.told((int)i) : -1;
      weights_out[i] = x;
      positions_out[i] = p;
    }
    return;
  }
  // the budget-th largest rank, eight bits at a time
  uint32_t prefix = 0;
  int need = a.budget;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < kBins * kCopies; i += kEvictThreads) (&bins[0][0])[i] = 0;
    block_sync();
    const uint32_t above = shift == 24 ? 0 : 0xffffffffu << (shift + 8);
#pragma unroll 4
    for (int i = tid; i < length; i += kEvictThreads) {
      const uint32_t r = row.rank(i);
      if ((r & above) == prefix) atomicAdd(&bins[r >> shift & 255][lane % kCopies], 1u);
    }
    block_sync();
    if (tid < kBins) {
      int sum = 0;
#pragma unroll 8
      for (int i = 0; i < kCopies; ++i) sum += (int)bins[tid][(i + tid) % kCopies];
      sums[tid] = sum;
    }
    block_sync();
    if (w == 0) {                        // lane i: digits 255 - 4 i .. 252 - 4 i
      int x[4], all = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) all += x[e] = sums[255 - 4 * lane - e];
      int before = all;
      for (int o = 1; o < kWave; o *= 2) {
        const int y = __shfl_up(before, o);
        if (lane >= o) before += y;
      }
      before -= all;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (before < need && need <= before + x[e]) {
          found[0] = 255 - 4 * lane - e;
          found[1] = need - before;
        }
        before += x[e];
      }
    }
    block_sync();
    prefix |= (uint32_t)found[0] << shift;
    need = found[1];
    block_sync();
  }
  // `need` of the tokens of rank `prefix` stay, the lowest slots; a wave counts a run of slots
  const int part = (((length + kEvictWaves - 1) / kEvictWaves) + kWave - 1) / kWave * kWave;
  const int begin = min(w * part, length), end = min(begin + part, length);
  int equal[2] = {0, 0}, over[2] = {0, 0};
  for (int i0 = begin; i0 < end; i0 += kWave) {
    const int i = i0 + lane;
    const uint32_t r = i < end ? row.rank(i) : 0;
    const bool here = i < end, low = i < a.budget;
    equal[0] += __popcll(__ballot(here && r == prefix && low));
    equal[1] += __popcll(__ballot(here && r == prefix && !low));
    over[0] += __popcll(__ballot(here && r > prefix && low));
    over[1] += __popcll(__ballot(here && r > prefix && !low));
  }
  if (lane == 0) {
    for (int e = 0; e < 2; ++e) {
      wave_equal[e][w] = equal[e];
      wave_above[e][w] = over[e];
    }
  }
  block_sync();
  // equal ones, free slots and moves before this wave's run; all moves
  int equals = 0, to = 0, from = 0, moves = 0, same_before = 0, kept_low = 0;
  for (int x = 0; x < kEvictWaves; ++x) {
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
  u32x2* list = a.moves + bh * a.room;
  const uint64_t below = (1ull << lane) - 1;
  for (int i0 = begin; i0 < end; i0 += kWave) {
    const int i = i0 + lane;
    const bool here = i < end, low = i < a.budget;
    const uint32_t r = here ? row.rank(i) : 0;
    const uint64_t same = __ballot(here && r == prefix);
    const bool kept = here && (r > prefix || (r == prefix && equals + __popcll(same & below) < need));
    const uint64_t holes = __ballot(here && !kept && low), far = __ballot(kept && !low);
    if (here && !kept && low) reinterpret_cast<uint32_t*>(list + to + __popcll(holes & below))[0] = i;
    if (kept && !low) reinterpret_cast<uint32_t*>(list + from + __popcll(far & below))[1] = i;
    if (kept && low) {
      const float x = row.weights[i];
      const int p = row.position(i);
      weights_out[i] = x;
      positions_out[i] = p;
    }
    equals += __popcll(same);
    to += __popcll(holes);
    from += __popcll(far);
  }
  if (tid == 0) a.counts[bh] = moves;
  __threadfence_block();
  block_sync();
  for (int i = tid; i < moves; i += kEvictThreads) {
    const u32x2 move = list[i];
    const float x = row.weights[move[1]];
    const int p = row.position((int)move[1]);
    weights_out[move[0]] = x;
    positions_out[move[0]] = p;
  }
  block_sync();                          // the outputs may be the inputs
  for (int64_t i = a.budget + tid; i < a.row; i += kEvictThreads) {
    weights_out[i] = 0.0f;
    positions_out[i] = -1;
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
  a.batch = cache->batch;
  a.budget = budget; a.recent = recent; a.sinks = sinks;
  a.room = (int)evict_room(*cache, budget);
  a.weights = weights; a.positions = positions; a.seen = seen;
  a.weights_out = weights_out; a.positions_out = positions_out; a.lengths_out = lengths_out;
  a.counts = static_cast<int32_t*>(workspace);
  a.moves = reinterpret_cast<u32x2*>(static_cast<uint8_t*>(workspace) + rows * 8);
  hipStream_t st = static_cast<hipStream_t>(stream);
  paged_evict_kernel<<<(unsigned)rows, kEvictThreads, 0, st>>>(a);
  const int launched = launch_status("paged_evict");
  if (launched != SPX_OK || budget >= (int64_t)cache->table_width * cache->page_size) return launched;
  MoveArgs m{};
  m.map = a.map;
  m.batch = a.batch;
  m.room = a.room;
  m.pages = PagePointers{cache->key_pages, cache->value_pages, cache->key_scales, cache->value_scales};
  m.counts = a.counts;
  m.moves = a.moves;
  return launch_moves(m, cache->head_dim, st);
}
