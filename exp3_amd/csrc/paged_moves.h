// Moves of rows within the paged cache, shared by the eviction's two parts.
#pragma once

#include "paged.h"

namespace spx {

struct PagePointers {
  void* keys;
  void* values;
  void* key_scales;
  void* value_scales;
};

constexpr int kMoveThreads = 256;

struct MoveArgs {
  PagedMap map;
  int batch, room;                       // room: of a list
  PagePointers pages;
  const int32_t* counts;                 // [B, Hkv] moves of each list
  const u32x2* moves;                    // [B, Hkv, room] (to, from)
  int64_t row;                           // elements of a row of weights and positions
  const int32_t* seen;                   // [B], or null: the old lengths, which the map's starts are
  const float* weights;                  // [B, Hkv, row]
  const int32_t* positions;              // the same, or null
  float* weights_out;                    // these may be those
  int32_t* positions_out;
};

int launch_moves(const MoveArgs& a, int head_dim, hipStream_t st);

}  // namespace spx
