// Attention over the 8-bit cache for few rows: a launch's shape, and the kernels for new tokens in a line.
#include "ktir_kv8_rows_dev.h"

namespace ktir {

// the launch's shape: columns in 64s (192 alone has its three: other heads' loads of 12 codes would pass their end), rows, splits
void kv8_rows_shape(const ktir_kv8_attn_t& d, KV8Shape* s) {
  const int D = (int)d.cache.columns;
  const int64_t grp = d.q_heads / d.cache.heads;
  s->J = D <= 64 ? 1 : D <= 128 ? 2 : D == 192 ? 3 : 4;
  s->MT = d.max_q * grp > 16 ? 2 : 1;
  const int64_t TM = 16 * s->MT;
  s->slots = d.max_q * grp > TM ? d.batch.tokens * grp / TM + d.batch.seqs : d.batch.seqs;
  s->rows = (int)(d.max_q * grp < TM ? d.max_q * grp : TM);
  if (s->rows < 1) s->rows = 1;
  s->part = s->rows * (64 * s->J + 4);
  // the most tokens that a tile's rows see, from a step's bound on
  s->span = d.max_k;
  const int64_t near = d.window + (TM - 1) / grp + 1;
  if (d.window && near < s->span) s->span = near;
  s->span += ROWS_STEP - 1;
  // Heads of a workgroup, parts of the keys.  Up to 2^19 keys (times KV heads) a wavefront's
  // four work on one head, on parts of 128 keys or more: one workgroup a CU is best for one
  // sequence (65536 tokens of 8 heads: 36.8 us, two a CU 42.5), four for several (8 of up
  // to 8192: 20.5, 28.6 with one).  More come from HBM, which gives 4.8 TB/s to 128-byte
  // rows of one head each, 5.6 where four heads' rows are read together (read patterns of
  // 268 MB; 64 sequences of 2460 tokens: 77 and 68.6 us).  There one workgroup a CU is
  // best for one sequence (131072 tokens: 59.5 us, two 62.6); several, whose lengths the
  // host does not know, get four if all were the longest, with parts of 512 keys or more
  // (64 of 64 to 8192 tokens: parts of 1056 keys 78 us, of 832 74, of 2080 100, of 416 95;
  // 64 of 2460: parts of 640 68 us, of 256 81; 256 of up to 2048: of 544 88, of 1056 94).
  const int64_t heads = d.cache.heads, longest = s->span - (ROWS_STEP - 1), keys = s->slots * heads * longest;
  const bool tiles = !one_tile(d, (int)TM, (int)grp), far = keys > (1 << 19) && !tiles;
  s->HW = !far ? 1 : heads % 4 == 0 ? 4 : heads % 2 == 0 ? 2 : 1;
  const int64_t sets = s->slots * heads / s->HW;
  int64_t n = sets ? (tiles || s->slots <= 1 ? 256 : 1024) / sets : 1;
  if (far && s->slots > 1) {
    const int64_t even = longest / 512;
    n = n < 4 ? 4 : n;
    n = n < even ? n : even;
  }
  const int64_t most = (s->span + 127) / 128;
  n = n > most ? most : n;
  s->splits = n < 1 ? 1 : n > MOST_SPLITS ? MOST_SPLITS : (int)n;
}

template <int CODE, int J>
static int launch_j(const ktir_kv8_attn_t& d, const KV8Shape& s) {
  return s.MT == 2 ? kv8_rows_go<CODE, J, 2, false>(d, {}, s) : kv8_rows_go<CODE, J, 1, false>(d, {}, s);
}

template <int CODE>
static int launch_code(const ktir_kv8_attn_t& d, const KV8Shape& s) {
  switch (s.J) {
    case 1: return launch_j<CODE, 1>(d, s);
    case 2: return launch_j<CODE, 2>(d, s);
    case 3: return launch_j<CODE, 3>(d, s);
    default: return launch_j<CODE, 4>(d, s);
  }
}

int kv8_rows_launch(const ktir_kv8_attn_t& d, const KV8Shape& s) {
  return d.cache.dtype == KTIR_I8 ? launch_code<KTIR_I8>(d, s) : launch_code<KTIR_E4M3>(d, s);
}

}  // namespace ktir
