// What the kernels of attention over a paged cache leave to the joins (paged_join.cu).
#pragma once

#include "common.cuh"
#include "paged.cuh"

namespace ib200 {

constexpr int HALF_ROWS = 128;             // query rows of half a tile of chunks

// Descriptions of the tile that begins in a CTA and ends in another (last_cta; -1: there is none)
struct RowsJoin {
  int last_cta;
  int row, head;           // first row of q of its sequence, key head
  int tile_row, rows;      // its first row among the sequence's, how many it has
  int sequence;
};
struct ChunkJoin {
  int last_cta;
  int row, head, tokens;   // first row of q, key head, tokens from there on in the sequence
  int sequence;
};
static_assert(sizeof(RowsJoin) <= kPagedEntry && sizeof(ChunkJoin) <= kPagedEntry, "room ahead of the parts");

}  // namespace ib200
