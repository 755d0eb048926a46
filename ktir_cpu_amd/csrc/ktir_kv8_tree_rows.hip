// Attention of drafted tokens over the 8-bit cache: the kernels for few rows.
#include "ktir_kv8_rows_dev.h"
#include "ktir_kv8_tree.h"

namespace ktir {

template <int CODE, int J>
static int tree_rows_j(const ktir_kv8_attn_t& d, const KV8Mask& mask, const KV8Shape& s) {
  return s.MT == 2 ? kv8_rows_go<CODE, J, 2, true>(d, mask, s) : kv8_rows_go<CODE, J, 1, true>(d, mask, s);
}

template <int CODE>
static int tree_rows_code(const ktir_kv8_attn_t& d, const KV8Mask& mask, const KV8Shape& s) {
  switch (s.J) {
    case 1: return tree_rows_j<CODE, 1>(d, mask, s);
    case 2: return tree_rows_j<CODE, 2>(d, mask, s);
    case 3: return tree_rows_j<CODE, 3>(d, mask, s);
    default: return tree_rows_j<CODE, 4>(d, mask, s);
  }
}

int tree_rows_launch(const ktir_kv8_attn_t& d, const KV8Mask& mask, const KV8Shape& s) {
  return d.cache.dtype == KTIR_I8 ? tree_rows_code<KTIR_I8>(d, mask, s) : tree_rows_code<KTIR_E4M3>(d, mask, s);
}

}  // namespace ktir
