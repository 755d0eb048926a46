// Attention of drafted tokens over the 8-bit cache: the entry points' checks and the choice of a kernel.
//
// A row sees the keys before its sequence's new ones, from its window on, and those new ones that its mask names.  Which of
// 32 keys a row sees is one word, of two of its mask's; before the new ones it is all ones and nothing is loaded for it, so the
// kernels are those of new tokens in a line (ktir_kv8_rows_dev.h, ktir_kv8_tile_dev.h) but for where a step reaches the
// window's start or the new tokens.  Their tiles' keys are cut by the device (ktir_kv8_dev.h), and a second kernel joins the parts.
//
// 32 / 8 heads of 128 columns, in loops of launches on inputs in turn; kernels under a profiler.  8 tokens after 1000: 12.6 us, latency (8.7 and
// 4.4 for the join).  64 sequences of up to 8 after 64 to 8192, 208 MB: 66, 55 at 3.8 TB/s and 12 for the join.  64 after 131072, 137
// GFLOP and half as many for the weights' second terms: 208 to 210, the products at 1.0 PFLOP/s (198) and 11 for the join; 252 for the first launches
// of an idle card.  8 of 128 to 256 after 2048 to 16384, 199 GFLOP and half as many: 376 to 382 (362 and 22; 443 for the first launches), an even share
// of the steps is 318.  12 of up to 100 after up to 4000, a window of 1000, 21 / 3 heads of 80: 31.5, the longest piece and a join (24 and 7).
#include "ktir_kv8_tree.h"

namespace ktir {

constexpr int64_t MASK_WORDS = 32;

struct TreePlan {
  bool tile;
  KV8Shape rows;       // tile false
  TreeTiles tiles;     // true
  int64_t groups, floats;       // how many share the keys of a head; of the workspace for each
};

// The kernels for few rows, MT tiles of 16 each.
static KV8Shape tree_rows(const ktir_kv8_attn_t& d, int MT, int64_t span) {
  const int64_t grp = d.q_heads / d.cache.heads, rows = d.max_q * grp, TM = 16 * MT;
  KV8Shape s = {};
  s.J = d.cache.columns <= 64 ? 1 : d.cache.columns <= 128 ? 2 : d.cache.columns == 192 ? 3 : 4;
  s.MT = MT;
  s.HW = 1;
  s.slots = rows > TM ? d.batch.tokens * grp / TM + d.batch.seqs : d.batch.seqs;
  s.rows = rows < 1 ? 1 : rows < TM ? (int)rows : (int)TM;
  s.part = s.rows * (64 * s.J + 4);
  s.span = span + 31;                    // (from a step's bound on)
  return s;
}

static TreePlan tree_plan(const ktir_kv8_attn_t& d) {
  TreePlan p = {};
  const int64_t heads = d.cache.heads, grp = d.q_heads / heads, rows = d.max_q * grp;
  const bool wide = d.cache.columns > 128;
  int64_t span = d.max_k;                // the most keys that a tile's rows see
  if (d.window && d.window + d.max_q < span) span = d.window + d.max_q;
  // Little work takes tiles of 16 rows, however many: more workgroups and shorter ones (eight KV heads of 128 columns, 4 query
  // heads each, one sequence: 8 tokens after 1000 13.2 us, tiles of 32 rows 15.7; 64 after 1000 19.0, of 256 27.3; 16 after
  // 16000 34.7, 29.6; sixteen sequences of 16 after 1000 38.6, 32.5).  Tiles of 32 rows read the cache half as often, but with more
  // than 128 columns leave a SIMD one wavefront, so that they need longer keys, or more work, where lengths are uneven (192 and 256
  // columns, tiles of 16 rows and of 32: four sequences of 16 tokens after 4000 46.7 and 60.3, 37.4 and 42.6; one after 16000 45.1 and
  // 58.3, 35.7 and 40.6; 14 after 200 to 1500 42.8 and 54.0, 64.4 and 73.1; 28 of four KV heads after 200 to 2000 39.5 and 49.9, 53.9 and
  // 59.0, after 1800 to 2000 60.2 and 85.5, 52.3 and 59.8; 20 of two after 300 to 5000 30.5 and 37.3, 33.6 and 37.2).  Up to 64 rows two tiles of 32 beat one of 256 (80 rows 57 us, 44;
  // 192 of six sequences 194, 142) and beat one of 64 by what that spills (64 rows of 16 sequences of up to 16000: 51, 69).
  const KV8Shape least = tree_rows(d, 1, span);
  const int64_t tiles = least.slots * heads;
  const bool little = tiles <= 512 && tiles * span <= 1 << 18;
  if (rows <= 64 || little) {
    const bool narrow = little || rows <= 16 || (wide && tiles <= 2048 && tiles * span <= 1 << 20 && span < 3500);
    KV8Shape& s = p.rows = narrow ? least : tree_rows(d, 2, span);
    const int64_t n = s.slots * heads, most = s.slots * ((s.span + 127) / 128);
    // Heads of a workgroup: several, a wavefront each, for many tiles of few keys, where nothing is left to join then (200
    // sequences of 8 tokens after up to 500: 56.7 us, a workgroup for each head 72; up to 2000 156, 151), and for many long ones, whose
    // rows of several heads are read together (one, two and four heads, of eight, 1 to 8 tokens: 64 sequences of 64 to 8192 keys 78.0, 69.1,
    // 68.9; 100 117.6, 137.3, 108.3; 64 of 64 to 4000 55.6, 48.0, 50.5; 128 116.8, 97.9, 105.4; 128 of four heads, 64 to 8192, 84.0, 85.4, 78.6;
    // where lengths are alike one or two gain: 128 of 1000 to 2500 123.8, 124.9, 143.3; 64 of 8 tokens after 2500 98.2, 95.2, 100.5).
    const bool many = n >= 1024 && span <= (wide ? 2048 : 768), far = n >= 512 && n < 2048 && span > 2048;
    if (many || far) s.HW = heads % 4 == 0 ? 4 : heads % 2 == 0 ? 2 : 1;
    // Parts that the device may cut: the workgroups that the chip holds, and two at least for each tile (eight sequences for each CU are not cut).
    const int64_t sets = heads / s.HW, held = kv8_rows_held(s.J, s.MT);
    int64_t parts = held / sets > 2 * s.slots ? held / sets : 2 * s.slots;
    if (parts > most) parts = most;
    p.groups = many || n >= 2048 || span <= tree_cut_cost(n) || parts <= s.slots ? 1 : parts;
    p.floats = heads * s.part;
    return p;
  }
  p.tile = true;
  TreeTiles& t = p.tiles;
  t.J = d.cache.columns <= 64 ? 1 : d.cache.columns <= 128 ? 2 : 4;
  t.TM = t.J == 4 || (t.J == 1 && rows <= 128) ? 128 : 256;
  t.slots = rows > t.TM ? d.batch.tokens * grp / t.TM + d.batch.seqs : d.batch.seqs;
  t.waves = (int)((rows < t.TM ? rows : t.TM) + 31) / 32;
  // Pieces that the device may cut: one for each CU where that cuts every tile into several; up to 1024 tiles two for each, so that no long
  // tile is left at the end (more give evener shares, but each costs 12 us and 264 KB to and from the workspace); more tiles
  // are not cut.  No more than the longest sequence can have.
  const int64_t n = t.slots * heads, most = t.slots * ((span / 64 + 1) / TREE_LEAST + 1);
  int64_t pieces = n <= 1024 && span > tree_cut_cost(n) ? 2 * t.slots : t.slots;
  if (n <= 256 && pieces > t.slots && pieces < 256 / heads) pieces = 256 / heads;
  if (pieces > most) pieces = most;
  t.pieces = (int)(pieces > t.slots ? pieces : t.slots);
  p.groups = t.pieces > t.slots ? t.pieces : 1;
  p.floats = heads * tree_part_size(t.J, t.waves);
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
  d->attn.splits = (int32_t)p.groups;
  d->attn.ws_bytes = p.groups > 1 ? p.groups * p.floats * 4 + d->attn.batch.seqs * (int64_t)sizeof(TreeNote) : 0;
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
  const int64_t slots = p.tile ? p.tiles.slots : p.rows.slots;
  if (splits > (1 << 16) || (splits > 1 && splits <= slots)) return set_error(KTIR_E_ARG, "%s: %lld splits of %lld tiles", ME, (long long)splits, (long long)slots);
  if ((slots + 8) * d->cache.heads > INT32_MAX || splits * d->cache.heads > INT32_MAX)
    return set_error(KTIR_E_UNSUPPORTED, "%s: %lld tiles of %lld heads in %lld splits", ME, (long long)slots, (long long)d->cache.heads, (long long)splits);
  if (splits > 1 && (!d->ws || (d->ws & 15) || (d->ws_bytes - d->batch.seqs * (int64_t)sizeof(TreeNote)) / 4 / p.floats < splits))
    return set_error(KTIR_E_ARG, "%s: %lld splits with a workspace of %lld bytes at %llx", ME, (long long)splits, (long long)d->ws_bytes, (unsigned long long)d->ws);
  rc = ready(ME);
  if (rc != KTIR_OK) return rc;
  OnDevice on;
  if (!on.ok()) return set_error(KTIR_E_HIP, "%s: no device", ME);
  const KV8Mask m = {t->mask, t->pos, t->mask_row, (int32_t)t->words, 0};
  if (!p.tile) return tree_rows_launch(*d, m, p.rows);
  p.tiles.pieces = splits > 1 ? (int)splits : (int)p.tiles.slots;
  return tree_tile_launch(*d, m, p.tiles);
}
