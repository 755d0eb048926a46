// Attention of drafted tokens over the 8-bit cache: the kernels for many rows.
#include "ktir_kv8_tile_dev.h"
#include "ktir_kv8_tree.h"

namespace ktir {

template <int CODE, int J, int W, bool IDLE = false>
static void tree_tile_go(const ktir_kv8_attn_t& d, const KV8Mask& mask, const TreeTiles& s) {
  const unsigned heads = (unsigned)d.cache.heads, items = (unsigned)s.slots * heads;
  const hipStream_t st = stream_of(d.stream);
  hipLaunchKernelGGL((kv8_attn_tile<CODE, J, 1, W, true, IDLE>), dim3(s.pieces * heads), dim3(64 * W), 0, st, d, mask, (uint32_t)s.slots, s.pieces, s.waves, device_error_flag());
  if (s.pieces > s.slots) {
    // many tiles: more for each wavefront, which has to find its place first
    constexpr int V = J == 1 ? 2 : 4;
    if (items <= 16) hipLaunchKernelGGL((kv8_tile_join<J, 1, 16>), dim3(items, s.waves, 2 * J), dim3(256), 0, st, d, s.pieces, s.waves, s.TM, device_error_flag());
    else hipLaunchKernelGGL((kv8_tile_join<J, V, 8>), dim3(items, s.waves, 2 * J / V), dim3(256), 0, st, d, s.pieces, s.waves, s.TM, device_error_flag());
  }
}

template <int CODE>
static void tree_tile_code(const ktir_kv8_attn_t& d, const KV8Mask& mask, const TreeTiles& s) {
  switch (s.J) {
    case 1: return s.TM == 128 ? tree_tile_go<CODE, 1, 4>(d, mask, s) : tree_tile_go<CODE, 1, 8>(d, mask, s);
    case 2: return s.waves <= 4 ? tree_tile_go<CODE, 2, 8, true>(d, mask, s) : tree_tile_go<CODE, 2, 8>(d, mask, s);
    default: return tree_tile_go<CODE, 4, 4>(d, mask, s);
  }
}

int tree_tile_launch(const ktir_kv8_attn_t& d, const KV8Mask& mask, const TreeTiles& s) {
  d.cache.dtype == KTIR_I8 ? tree_tile_code<KTIR_I8>(d, mask, s) : tree_tile_code<KTIR_E4M3>(d, mask, s);
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}

}  // namespace ktir
