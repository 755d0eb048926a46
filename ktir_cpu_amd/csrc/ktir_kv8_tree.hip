// Attention of drafted tokens over the 8-bit cache: the entry points' checks and the choice of a kernel.
#include "ktir_kv8_tree.h"

namespace ktir {

constexpr int64_t MASK_WORDS = 32;

// Whether a launch's rows of a KV head are more than one tile of the kernels for few rows takes.
static bool tree_tiles(const ktir_kv8_attn_t& d, const KV8Shape& s) { return d.max_q * (d.q_heads / d.cache.heads) > 16 * s.MT; }

struct TreePlan {
  bool tile;
  KV8Shape rows;       // tile false
  TreeTiles tiles;     // true
  int64_t items, floats;        // tiles of rows times KV heads; of a split's part
};

static TreePlan tree_plan(const ktir_kv8_attn_t& d) {
  TreePlan p = {};
  kv8_rows_shape(d, true, &p.rows);
  p.tile = tree_tiles(d, p.rows);
  if (p.tile) {
    const int64_t grp = d.q_heads / d.cache.heads, most = d.max_q * grp;
    TreeTiles& t = p.tiles;
    t.J = d.cache.columns <= 64 ? 1 : d.cache.columns <= 128 ? 2 : 4;
    t.TM = t.J == 4 ? 128 : 256;
    t.slots = most > t.TM ? d.batch.tokens * grp / t.TM + d.batch.seqs : d.batch.seqs;
    t.waves = (int)((most < t.TM ? most : t.TM) + 31) / 32;
    t.span = d.max_k;
    if (d.window && d.window + d.max_q < t.span) t.span = d.window + d.max_q;
    t.span += 63;
    const int64_t sets = t.slots * d.cache.heads;
    int64_t n = sets ? 256 / sets : 1;
    const int64_t most_parts = (t.span + 255) / 256;
    n = n > most_parts ? most_parts : n;
    t.splits = n < 1 ? 1 : n > 256 ? 256 : (int)n;
    p.items = sets;
    p.floats = (int64_t)t.waves * (2048 * t.J + 64);
  } else {
    p.items = p.rows.slots * d.cache.heads;
    p.floats = p.rows.part;
  }
  return p;
}

static int check_tree(const char* what, const ktir_kv8_tree_attn_t& t) {
  const int rc = check_kv8_attn(what, t.attn, true);
  if (rc != KTIR_OK) return rc;
  if (t.words < 1 || t.words > MASK_WORDS) return set_error(KTIR_E_UNSUPPORTED, "%s: masks of %lld words (1 to %lld)", what, (long long)t.words, (long long)MASK_WORDS);
  if (t.attn.max_q > 32 * t.words) return set_error(KTIR_E_ARG, "%s: %lld new tokens, masks of %lld words", what, (long long)t.attn.max_q, (long long)t.words);
  if (t.mask_row < 0 || t.mask_row > ((int64_t)1 << 40)) return set_error(KTIR_E_ARG, "%s: mask stride %lld", what, (long long)t.mask_row);
  return KTIR_OK;
}

}  // namespace ktir

using namespace ktir;

extern "C" int ktir_kv8_tree_attention_plan(ktir_kv8_tree_attn_t* d) {
  constexpr const char* ME = "ktir_kv8_tree_attention_plan";
  if (!d) return set_error(KTIR_E_ARG, "%s: no descriptor", ME);
  const int rc = check_tree(ME, *d);
  if (rc != KTIR_OK) return rc;
  const TreePlan p = tree_plan(d->attn);
  d->attn.splits = p.tile ? p.tiles.splits : p.rows.splits;
  d->attn.ws_bytes = d->attn.splits > 1 ? p.items * d->attn.splits * p.floats * 4 : 0;
  return KTIR_OK;
}

extern "C" int ktir_launch_kv8_tree_attention(const ktir_kv8_tree_attn_t* t) {
  constexpr const char* ME = "ktir_launch_kv8_tree_attention";
  if (!t) return set_error(KTIR_E_ARG, "%s: no descriptor", ME);
  int rc = check_tree(ME, *t);
  const ktir_kv8_attn_t* d = &t->attn;
  if (rc != KTIR_OK || d->batch.seqs == 0 || d->batch.tokens == 0) return rc;
  if (!t->mask || ((t->mask | t->pos) & 3) || (d->window && !t->pos)) return set_error(KTIR_E_ARG, "%s: mask or positions missing or off 4-byte bounds", ME);
  rc = check_kv8_attn_tensors(ME, *d);
  if (rc != KTIR_OK) return rc;
  const Strided mask(t->mask, t->words * 4, d->batch.tokens, t->mask_row * 4), pos = t->pos ? Strided(t->pos, d->batch.tokens * 4) : mask;
  const Strided out = rows_of(d->out, d->batch.tokens, d->q_heads, d->cache.columns, 2), lse = rows_of({d->lse, d->lse_tok, d->lse_head}, d->batch.tokens, d->q_heads, 1, 4);
  const Strided ws = d->splits > 1 && d->ws && d->ws_bytes > 0 ? Strided(d->ws, d->ws_bytes) : out;
  if (!apart(out, mask) || !apart(out, pos) || !apart(ws, mask) || !apart(ws, pos) || (d->lse && (!apart(lse, mask) || !apart(lse, pos))))
    return set_error(KTIR_E_ARG, "%s: an output or the workspace overlaps the mask or positions", ME);
  TreePlan p = tree_plan(*d);
  const int64_t splits = d->splits < 1 ? 1 : d->splits;
  if (splits > 256) return set_error(KTIR_E_ARG, "%s: %lld splits, 256 at most", ME, (long long)splits);
  if (p.items > INT32_MAX / splits) return set_error(KTIR_E_UNSUPPORTED, "%s: %lld tiles in %lld splits", ME, (long long)p.items, (long long)splits);
  if (splits > 1 && (!d->ws || (d->ws & 15) || d->ws_bytes / 4 / p.floats / p.items < splits))
    return set_error(KTIR_E_ARG, "%s: %lld splits with a workspace of %lld bytes at %llx", ME, (long long)splits, (long long)d->ws_bytes, (unsigned long long)d->ws);
  rc = ready(ME);
  if (rc != KTIR_OK) return rc;
  OnDevice on;
  if (!on.ok()) return set_error(KTIR_E_HIP, "%s: no device", ME);
  const KV8Mask m = {t->mask, t->pos, t->mask_row, (int32_t)t->words, 0};
  if (!p.tile) return tree_rows_launch(*d, m, p.rows);
  p.tiles.splits = (int)splits;
  return tree_tile_launch(*d, m, p.tiles);
}
