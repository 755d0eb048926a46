// What the files of the attention of drafted tokens share.
#pragma once
#include "ktir_kv8_dev.h"

namespace ktir {

constexpr int TREE_LEAST = 4;          // steps of 64 keys that a piece of a tile has at least

// Floats that a piece leaves in the workspace, of so many wavefronts: they lie as the lanes have them, 8 J vectors of 4
// columns of each wavefront's 64 lanes, then b and l of 32 rows.
__host__ __device__ constexpr int64_t tree_part_size(int J, int waves) { return (int64_t)waves * (32 * 64 * J + 64); }

// The shape of a launch of ktir_kv8_tree_tile.hip.
struct TreeTiles {
  int J, TM, waves, pieces;      // columns in 64s (1, 2, 4), rows of a tile, wavefronts that have rows, pieces of a head (its tiles: none is cut)
  int64_t slots;                 // tiles of rows for each KV head
};

int tree_rows_launch(const ktir_kv8_attn_t& d, const KV8Mask& mask, const KV8Shape& s);
int tree_tile_launch(const ktir_kv8_attn_t& d, const KV8Mask& mask, const TreeTiles& s);

}  // namespace ktir
