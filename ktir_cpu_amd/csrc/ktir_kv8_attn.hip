// Attention over the key / value cache in 8 bits: the entry points' checks and
// the choice of a kernel.
#include "ktir_serve.h"

namespace ktir {

int check_kv8_attn(const char* what, const ktir_kv8_attn_t& d, bool tree) {
  if (d.dtype != KTIR_F16 && d.dtype != KTIR_BF16) return set_error(KTIR_E_UNSUPPORTED, "%s: dtype %d", what, d.dtype);
  int rc = check_kv8(what, d.cache, false);
  if (rc == KTIR_OK) rc = check_batch(what, d.batch, d.cache);
  if (rc != KTIR_OK) return rc;
  if (d.q_heads < 1 || d.q_heads % d.cache.heads || d.q_heads > 65536)
    return set_error(KTIR_E_ARG, "%s: %lld query heads over %lld", what, (long long)d.q_heads, (long long)d.cache.heads);
  if (d.max_q < 0 || d.max_q > INT32_MAX || d.max_k < 0 || d.max_k > (1 << 30)) return set_error(KTIR_E_ARG, "%s: bounds %lld and %lld", what, (long long)d.max_q, (long long)d.max_k);
  if (d.window < 0 || d.window > INT32_MAX || (d.window && !d.causal && !tree)) return set_error(KTIR_E_ARG, "%s: window %lld", what, (long long)d.window);
  if (!(d.scale - d.scale == 0.f)) return set_error(KTIR_E_ARG, "%s: scale is not finite", what);
  if (d.batch.tokens * (d.q_heads / d.cache.heads) > (1 << 30)) return set_error(KTIR_E_UNSUPPORTED, "%s: %lld rows of a KV head", what, (long long)(d.batch.tokens * (d.q_heads / d.cache.heads)));
  if (d.splits < 0) return set_error(KTIR_E_ARG, "%s: %d splits", what, d.splits);
  return KTIR_OK;
}

// q, out, lse and the workspace: strides, and that what is written shares no byte with anything else
int check_kv8_attn_tensors(const char* what, const ktir_kv8_attn_t& d) {
  int rc = check_rows3(what, d.q, d.batch.tokens, d.q_heads, d.cache.columns, false);
  if (rc == KTIR_OK) rc = check_rows3(what, d.out, d.batch.tokens, d.q_heads, d.cache.columns, true);
  if (rc == KTIR_OK && d.lse) {
    rc = d.lse & 3 ? set_error(KTIR_E_ARG, "%s: lse off 4-byte bounds", what)
                    : check_rows3(what, {d.lse, d.lse_tok, d.lse_head}, d.batch.tokens, d.q_heads, 1, true);
  }
  if (rc != KTIR_OK) return rc;
  auto rows = [&](const ktir_rows3_t& r, int64_t columns, int64_t bytes) { return rows_of(r, d.batch.tokens, d.q_heads, columns, bytes); };
  const Strided q = rows(d.q, d.cache.columns, 2), out = rows(d.out, d.cache.columns, 2);
  const Strided lse = rows({d.lse, d.lse_tok, d.lse_head}, 1, 4);
  if (!(same(q, out) || apart(q, out)) || (d.lse && !(apart(lse, out) && apart(lse, q))))
    return set_error(KTIR_E_ARG, "%s: an output overlaps a tensor that it is not", what);
  const CacheParts cache(d.cache);
  const BatchParts batch(d.batch);
  auto clear = [&](const Strided& x) { return apart(x, cache.x[0]) && apart(x, cache.x[1]) && apart(x, cache.x[2]) && apart(x, cache.x[3]) && batch.clear_of(x); };
  if (!clear(out) || (d.lse && !clear(lse))) return set_error(KTIR_E_ARG, "%s: an output overlaps the cache, table, offsets or lengths", what);
  if (d.splits > 1 && d.ws && d.ws_bytes > 0) {
    const Strided ws(d.ws, d.ws_bytes);
    if (!clear(ws) || !apart(out, ws) || !apart(q, ws) || (d.lse && !apart(lse, ws)))
      return set_error(KTIR_E_ARG, "%s: the workspace overlaps a tensor", what);
  }
  return KTIR_OK;
}

}  // namespace ktir

using namespace ktir;

extern "C" int ktir_kv8_attention_plan(ktir_kv8_attn_t* d) {
  constexpr const char* ME = "ktir_kv8_attention_plan";
  if (!d) return set_error(KTIR_E_ARG, "%s: no descriptor", ME);
  const int rc = check_kv8_attn(ME, *d, false);
  if (rc != KTIR_OK) return rc;
  KV8Shape s;
  int64_t slots;
  kv8_rows_shape(*d, &s);
  if (kv8_tile_takes(*d, &slots)) s.splits = 1;
  d->splits = s.splits;
  d->ws_bytes = s.splits > 1 ? s.slots * d->cache.heads * s.splits * s.part * 4 : 0;
  return KTIR_OK;
}

extern "C" int ktir_launch_kv8_attention(const ktir_kv8_attn_t* d) {
  constexpr const char* ME = "ktir_launch_kv8_attention";
  if (!d) return set_error(KTIR_E_ARG, "%s: no descriptor", ME);
  int rc = check_kv8_attn(ME, *d, false);
  if (rc != KTIR_OK || d->batch.seqs == 0 || d->batch.tokens == 0) return rc;
  rc = check_kv8_attn_tensors(ME, *d);
  if (rc != KTIR_OK) return rc;
  KV8Shape s;
  kv8_rows_shape(*d, &s);
  const int64_t splits = d->splits < 1 ? 1 : d->splits, tiles = s.slots * d->cache.heads;
  if (splits > 256) return set_error(KTIR_E_ARG, "%s: %lld splits, 256 at most", ME, (long long)splits);
  if (tiles > INT32_MAX / splits)
    return set_error(KTIR_E_UNSUPPORTED, "%s: %lld tiles in %lld splits", ME, (long long)tiles, (long long)splits);
  if (splits > 1 && (!d->ws || (d->ws & 15) || d->ws_bytes / 4 / s.part / tiles < splits))
    return set_error(KTIR_E_ARG, "%s: %lld splits with a workspace of %lld bytes at %llx", ME, (long long)splits, (long long)d->ws_bytes,
                     (unsigned long long)d->ws);
  rc = ready(ME);
  if (rc != KTIR_OK) return rc;
  OnDevice on;
  if (!on.ok()) return set_error(KTIR_E_HIP, "%s: no device", ME);
  int64_t slots;
  if (kv8_tile_takes(*d, &slots)) return kv8_tile_launch(*d, slots);
  return kv8_rows_launch(*d, s);
}
