// What the files of the attention of drafted tokens share.
#pragma once
#include "ktir_kv8_dev.h"

namespace ktir {

// The shape of a launch of ktir_kv8_tree_tile.hip.
struct TreeTiles {
  int J, TM, waves, splits;      // columns in 64s (1, 2, 4), rows of a tile, wavefronts that have rows, parts of the keys
  int64_t slots, span;           // tiles of rows for each KV head, most keys of a tile
};

int tree_rows_launch(const ktir_kv8_attn_t& d, const KV8Mask& mask, const KV8Shape& s);
int tree_tile_launch(const ktir_kv8_attn_t& d, const KV8Mask& mask, const TreeTiles& s);

}  // namespace ktir
