// Host side of the paged cache's tensor maps.
#pragma once

#include <cuda.h>

#include "paged.h"

namespace mlora {

// Rows of a TMA box: the largest power of two that divides both the block
// size and the key tile, so that no box leaves its block and boxes fill a tile.
inline int paged_box(int block_size, int tile) {
  const int low = block_size & -block_size;
  return low < tile ? low : tile;
}

// Maps {dim, slot, head, block} over K and V, box 64 columns x `box` slots,
// 128-byte swizzle, zeros out of range. False where a map cannot describe the cache.
bool paged_maps(const PagedAttnArgs& a, int dtype, int box, CUtensorMap* k, CUtensorMap* v);

// Map {dim, head, token} over Q, box 64 columns x group heads x rows / group tokens: a
// tile of `rows` packed rows (token major, then head). False where group does not divide it.
bool paged_q_map(const PagedAttnArgs& a, int dtype, int rows, CUtensorMap* q);

}  // namespace mlora
