// Rows of the paged cache moved within it: the accepted path of a tree of drafted tokens into
// place, and the tokens that an eviction keeps into the room of those that it drops.
//
// Bound by latencies (tree, path, page ids, rows; a wave per cache, K or V, and head walks the tree by
// itself): 16 nodes in 28 caches of 4 heads 3.8 us, 64 trees of 61 nodes in 12 caches of 8 heads 10.2 us,
// a given path 8.0, pages of 4 bits as long; one launch for 32 caches, where one each would be 28 launches.
#include <algorithm>

#include "paged_moves.h"

namespace spx {

// A lane's 16 bytes (and scales) of a row of K or V.
template <int D, bool kFour>
struct RowPart {
  static constexpr int kBytes = kFour ? D / 2 : 2 * D, kLanes = kBytes / 16, kRows = kWave / kLanes;
  static constexpr int kScales = D / kPagedGroup;
  u32x4 data;
  uint32_t scale;                        // four scale bytes: lanes below kScales / 4
  __device__ __forceinline__ void load(const uint8_t* pages, const uint8_t* scales, int64_t row,
                                       int piece) {
    data = *reinterpret_cast<const u32x4*>(pages + row * kBytes + 16 * piece);
    if (kFour && piece < kScales / 4)
      scale = *reinterpret_cast<const uint32_t*>(scales + row * kScales + 4 * piece);
  }
  __device__ __forceinline__ void store(uint8_t* pages, uint8_t* scales, int64_t row,
                                        int piece) const {
    *reinterpret_cast<u32x4*>(pages + row * kBytes + 16 * piece) = data;
    if (kFour && piece < kScales / 4)
      *reinterpret_cast<uint32_t*>(scales + row * kScales + 4 * piece) = scale;
  }
};

// ------------------------------------------------------------------------- paths

constexpr int kPathTokens = 256, kPathChunks = kPathTokens / kWave;
constexpr int kPathCaches = 32;          // of a launch
constexpr int kPathThreads = 256;

struct PathArgs {
  PagedMap map;
  int batch, tokens, caches;
  const int32_t* parents;                // [B, T]; null: the path is given
  const int64_t* drafts;
  const int64_t* targets;
  const int32_t* given;                  // [B, T]
  int32_t* accepted;                     // [B], or null
  int32_t* path;                         // [B, T]
  int64_t* following;                    // [B]
  PagePointers pages[kPathCaches];
};

// Element i of a [T] row that a wave holds, 64 a register.
template <typename T>
__device__ __forceinline__ T element(const T (&x)[kPathChunks], int i) {
  T out = 0;
#pragma unroll
  for (int n = 0; n < kPathChunks; ++n)
    if (i / kWave == n) {
      if constexpr (sizeof(T) == 8)
        out = (T)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)x[n], i % kWave) |
                  (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x[n] >> 32), i % kWave) << 32);
      else
        out = __builtin_amdgcn_readlane(x[n], i % kWave);
    }
  return out;
}

// One wave per (sequence, cache, K or V, head): finds the path by itself, then moves its rows, the
// first first: row j comes from one at or behind it, so what a later step reads is not written yet.
template <int D, bool kFour>
__global__ __launch_bounds__(kPathThreads) void paged_path_kernel(PathArgs a, int64_t items) {
  using Part = RowPart<D, kFour>;
  const int lane = threadIdx.x & 63;
  const int64_t first = (int64_t)blockIdx.x * (kPathThreads / kWave) +
                        __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  for (int64_t item = first; item < items; item += (int64_t)gridDim.x * (kPathThreads / kWave)) {
    const int head = (int)(item % a.map.kv_heads);
    const int64_t rest = item / a.map.kv_heads;
    const bool values = rest % 2 != 0;
    const int cache = (int)(rest / 2 % a.caches), b = (int)(rest / 2 / a.caches);
    const int start = a.map.starts[b], count = a.map.counts ? a.map.counts[b] : a.tokens;
    const int64_t room = a.map.capacity() - start;
    const int live = start < 0 ? 0
                               : max(0, min(min(count, a.tokens), (int)min(room, (int64_t)a.tokens)));
    const int64_t row0 = (int64_t)b * a.tokens;
    int path[kPathChunks];
#pragma unroll
    for (int n = 0; n < kPathChunks; ++n) path[n] = -1;
    int taken = 0;
    int64_t following = -1;
    if (a.parents != nullptr) {
      int parent[kPathChunks];
      int64_t draft[kPathChunks], target[kPathChunks];
#pragma unroll
      for (int n = 0; n < kPathChunks; ++n) {
        const int i = n * kWave + lane;
        const bool here = i < live;
        parent[n] = here ? a.parents[row0 + i] : -1;
        if (parent[n] >= i) parent[n] = -1;
        draft[n] = here ? a.drafts[row0 + i] : 0;
        target[n] = here ? a.targets[row0 + i] : 0;
      }
      int at = live > 0 ? 0 : -1;
      while (at >= 0) {                  // `at` grows: a child is behind its parent
#pragma unroll
        for (int n = 0; n < kPathChunks; ++n)
          if (n * kWave + lane == taken) path[n] = at;
        ++taken;
        following = element(target, at);
        int child = -1;
#pragma unroll
        for (int n = kPathChunks - 1; n >= 0; --n) {
          const uint64_t hit = __ballot(parent[n] == at && draft[n] == following);
          if (hit) child = n * kWave + __builtin_ctzll(hit);
        }
        at = child;
      }
    } else {
      int before = -1;
#pragma unroll
      for (int n = 0; n < kPathChunks; ++n) {
        const int j = n * kWave + lane;
        if (j < live) path[n] = a.given[row0 + j];
        const int prior = __shfl_up(path[n], 1);
        const bool good = path[n] < live && path[n] > (lane == 0 ? before : prior);
        const uint64_t wrong = ~__ballot(good);
        if (taken == n * kWave) taken += wrong ? __builtin_ctzll(wrong) : kWave;
        before = __builtin_amdgcn_readlane(path[n], kWave - 1);
      }
    }
    if (a.accepted != nullptr && rest % (2 * a.caches) == 0 && head == 0) {
      if (lane == 0) {
        a.accepted[b] = taken;
        a.following[b] = following;
      }
#pragma unroll
      for (int n = 0; n < kPathChunks; ++n)
        if (n * kWave + lane < a.tokens) a.path[row0 + n * kWave + lane] = path[n];
    }
    const PagePointers& to = a.pages[cache];
    uint8_t* pages = static_cast<uint8_t*>(values ? to.values : to.keys);
    uint8_t* scales = static_cast<uint8_t*>(values ? to.value_scales : to.key_scales);
    const int piece = lane % Part::kLanes;
    for (int j0 = 0; j0 < taken; j0 += Part::kRows) {
      const int j = j0 + lane / Part::kLanes;
      int from = 0;
#pragma unroll
      for (int n = 0; n < kPathChunks; ++n) {
        const int x = __shfl(path[n], j % kWave);
        if (j / kWave == n) from = x;
      }
      const bool moves = j < taken && from > j;
      const int source = moves ? a.map.page(b, start + from) : -1;
      const int target = moves ? a.map.page(b, start + j) : -1;
      if (source < 0 || target < 0) continue;
      Part part;
      part.load(pages, scales, a.map.row(source, head, start + from), piece);
      part.store(pages, scales, a.map.row(target, head, start + j), piece);
    }
  }
}

// ---------------------------------------------------------------------- evictions

// The tokens of the list of each (sequence, head) moved, from the second slot to the first, and the
// ledger cleared behind the old length.
template <int D, bool kFour>
__global__ __launch_bounds__(kMoveThreads) void paged_move_kernel(MoveArgs a) {
  using Part = RowPart<D, kFour>;
  constexpr int kAtOnce = 2;
  const int lane = threadIdx.x & 63, piece = lane % Part::kLanes;
  const int step = gridDim.x * (kMoveThreads / kWave) * Part::kRows;
  const int first = (blockIdx.x * (kMoveThreads / kWave) + threadIdx.x / kWave) * Part::kRows +
                    lane / Part::kLanes;
  uint8_t* const keys = static_cast<uint8_t*>(a.pages.keys);
  uint8_t* const values = static_cast<uint8_t*>(a.pages.values);
  uint8_t* const key_scales = static_cast<uint8_t*>(a.pages.key_scales);
  uint8_t* const value_scales = static_cast<uint8_t*>(a.pages.value_scales);
  for (int64_t bh = blockIdx.y; bh < (int64_t)a.batch * a.map.kv_heads; bh += gridDim.y) {
    const int b = (int)(bh / a.map.kv_heads), head = (int)(bh % a.map.kv_heads);
    const int count = min(a.counts[bh], a.room);
    const u32x2* list = a.moves + bh * a.room;
    const int length = a.map.starts[b], text = a.seen ? a.seen[b] : length;
    for (int64_t i = max(length, 0) + blockIdx.x * kMoveThreads + threadIdx.x; i < a.row;
         i += gridDim.x * kMoveThreads) {
      a.weights_out[bh * a.row + i] = 0.0f;
      a.positions_out[bh * a.row + i] = -1;
    }
    for (int i0 = first; i0 < count; i0 += kAtOnce * step) {
      Part k[kAtOnce], v[kAtOnce];
      int64_t to[kAtOnce];
      u32x2 move[kAtOnce];
      float weight[kAtOnce];
      int told[kAtOnce];
#pragma unroll
      for (int n = 0; n < kAtOnce; ++n) {
        move[n] = list[min(i0 + n * step, count - 1)];
        to[n] = a.map.row(max(a.map.page(b, (int)move[n][0]), 0), head, (int)move[n][0]);
        const int64_t from = a.map.row(max(a.map.page(b, (int)move[n][1]), 0), head, (int)move[n][1]);
        weight[n] = a.weights[bh * a.row + move[n][1]];
        told[n] = a.positions ? a.positions[bh * a.row + move[n][1]] : -1;
        k[n].load(keys, key_scales, from, piece);
        v[n].load(values, value_scales, from, piece);
      }
#pragma unroll
      for (int n = 0; n < kAtOnce; ++n) {
        if (i0 + n * step >= count) break;
        k[n].store(keys, key_scales, to[n], piece);
        v[n].store(values, value_scales, to[n], piece);
        if (piece == 0) {
          a.weights_out[bh * a.row + move[n][0]] = weight[n];
          a.positions_out[bh * a.row + move[n][0]] =
              told[n] >= 0 ? told[n] : text - length + (int)move[n][1];
          a.weights_out[bh * a.row + move[n][1]] = 0.0f;
          a.positions_out[bh * a.row + move[n][1]] = -1;
        }
      }
    }
  }
}

int launch_moves(const MoveArgs& a, int head_dim, hipStream_t st) {
  const bool four = a.pages.key_scales != nullptr;
  const int64_t rows = (int64_t)a.batch * a.map.kv_heads;
  const int per_block = kMoveThreads / kWave * 4;
  const int64_t most = std::max<int64_t>(1, 4096 / rows);
  const int64_t clears = (a.row + 8 * kMoveThreads - 1) / (8 * kMoveThreads);
  const dim3 grid((unsigned)std::min<int64_t>(most, std::max<int64_t>(clears, (a.room + per_block - 1) / per_block)),
                  (unsigned)std::min<int64_t>(rows, 65535));
  if (head_dim == 128) {
    if (four) paged_move_kernel<128, true><<<grid, kMoveThreads, 0, st>>>(a);
    else paged_move_kernel<128, false><<<grid, kMoveThreads, 0, st>>>(a);
  } else {
    if (four) paged_move_kernel<256, true><<<grid, kMoveThreads, 0, st>>>(a);
    else paged_move_kernel<256, false><<<grid, kMoveThreads, 0, st>>>(a);
  }
  return launch_status("paged_evict");
}

}  // namespace spx

using namespace spx;

extern "C" int spx_paged_keep_path(const spx_paged_cache* caches, int cache_count,
                                   const int32_t* parents, const int64_t* drafts,
                                   const int64_t* targets, const int32_t* path_in, int32_t* accepted,
                                   int32_t* path_out, int64_t* following, void* stream) {
  SPX_REQUIRE(caches && cache_count > 0, SPX_EINVAL, "no caches");
  PathArgs a{};
  const spx_paged_cache& first = caches[0];
  for (int i = 0; i < cache_count; ++i) {
    const spx_paged_cache& z = caches[i];
    const int status = paged_map(a.map, &z);
    if (status != SPX_OK) return status;
    SPX_REQUIRE(z.page_table == first.page_table && z.starts == first.starts &&
                    z.counts == first.counts && z.table_stride == first.table_stride &&
                    z.table_width == first.table_width && z.pages == first.pages &&
                    z.page_size == first.page_size && z.kv_heads == first.kv_heads &&
                    z.head_dim == first.head_dim && z.batch == first.batch &&
                    z.tokens == first.tokens &&
                    (z.key_scales == nullptr) == (first.key_scales == nullptr),
                SPX_EINVAL, "cache %d differs in more than its pages from the first", i);
    // rows would move twice, the second time from places that the first has filled
    for (int j = 0; j < i; ++j)
      SPX_REQUIRE(z.key_pages != caches[j].key_pages && z.value_pages != caches[j].value_pages,
                  SPX_EINVAL, "caches %d and %d are the same pages", j, i);
  }
  SPX_REQUIRE(first.tokens <= kPathTokens, SPX_EINVAL, "%d tokens are more than %d", first.tokens,
              kPathTokens);
  const bool walk = parents != nullptr;
  SPX_REQUIRE(walk == (drafts != nullptr) && walk == (targets != nullptr) &&
                  walk == (path_in == nullptr) && walk == (accepted != nullptr) &&
                  walk == (path_out != nullptr) && walk == (following != nullptr),
              SPX_EINVAL, "either parents, drafts, targets and the outputs, or path_in alone");
  SPX_REQUIRE(((reinterpret_cast<uintptr_t>(parents) | reinterpret_cast<uintptr_t>(path_in) |
                reinterpret_cast<uintptr_t>(accepted) | reinterpret_cast<uintptr_t>(path_out)) & 3) == 0 &&
                  ((reinterpret_cast<uintptr_t>(drafts) | reinterpret_cast<uintptr_t>(targets) |
                    reinterpret_cast<uintptr_t>(following)) & 7) == 0,
              SPX_EINVAL, "drafts, targets and following must be 8-byte, the others 4-byte aligned");
  a.batch = first.batch;
  a.tokens = first.tokens;
  a.parents = parents; a.drafts = drafts; a.targets = targets; a.given = path_in;
  a.accepted = accepted; a.path = path_out; a.following = following;
  const bool four = first.key_scales != nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  for (int done = 0; done < cache_count; done += kPathCaches) {
    a.caches = std::min(kPathCaches, cache_count - done);
    for (int i = 0; i < a.caches; ++i) {
      const spx_paged_cache& z = caches[done + i];
      a.pages[i] = PagePointers{z.key_pages, z.value_pages, z.key_scales, z.value_scales};
    }
    const int64_t items = (int64_t)a.batch * a.caches * 2 * first.kv_heads;
    const unsigned grid = (unsigned)std::min<int64_t>((items + 3) / 4, 1 << 22);
    if (first.head_dim == 128) {
      if (four) paged_path_kernel<128, true><<<grid, kPathThreads, 0, st>>>(a, items);
      else paged_path_kernel<128, false><<<grid, kPathThreads, 0, st>>>(a, items);
    } else {
      if (four) paged_path_kernel<256, true><<<grid, kPathThreads, 0, st>>>(a, items);
      else paged_path_kernel<256, false><<<grid, kPathThreads, 0, st>>>(a, items);
    }
    const int status = launch_status("paged_keep_path");
    if (status != SPX_OK) return status;
    a.accepted = nullptr;                // the first launch has written them
  }
  return SPX_OK;
}
