// Drafted tokens: positions and ancestor masks of a tree, and the accepted path's
// entries of the 8-bit cache.
#include "ktir_kv8_codes.h"

namespace ktir {

constexpr int64_t TREE_WORDS = 32;           // of a token's mask

// ---- the tree ----------------------------------------------------------------

// One thread a token: up its line of parents, bits from the highest word down.
__global__ __launch_bounds__(256) void draft_tree(const ktir_draft_tree_t d, int* err) {
  const int64_t s = blockIdx.x;
  const int64_t a = ints(d.q_start)[s], e = ints(d.q_start)[s + 1];
  const int64_t start = a < 0 ? 0 : a < d.tokens ? a : d.tokens, end = e < start ? start : e < d.tokens ? e : d.tokens;
  const int n = (int)(end - start), kv = ints(d.kv_len)[s], before = (kv < 0 ? 0 : kv) - n;
  if (start != a || end != e || kv < 0 || n > 32 * d.words) {
    *err = OUT_OF_RANGE;
    if (n > 32 * d.words) return;
  }
  const KTIR_G(int32_t)* parents = ints(d.parents) + start;
  for (int i = (int)(blockIdx.y * 256 + threadIdx.x); i < n; i += 256 * gridDim.y) {
    KTIR_G(uint32_t)* row = (KTIR_G(uint32_t)*)d.mask + (start + i) * d.mask_row;
    int j = i, depth = 0;
    for (int w = (int)d.words - 1; w >= 0; --w) {
      uint32_t bits = 0;
      while (j >= 32 * w) {
        if (!d.window || depth < d.window) bits |= 1u << (j & 31);
        const int p = parents[j];
        if (p < -1 || p >= j) *err = OUT_OF_RANGE;
        j = p < -1 || p >= j ? -1 : p;
        ++depth;
      }
      row[w] = bits;
    }
    ((KTIR_G(int32_t)*)d.positions)[start + i] = before + depth - 1;
  }
}

// ---- the kept path -----------------------------------------------------------

// One wavefront for a sequence, a KV head, and K or V.  Entries only move down and in order, so what a
// page gets is read before its place is written: pages in order, and in a page the rows of
// one pass of the wavefront (64 units of 16 columns), all read, then written.
template <int CODE>
__global__ __launch_bounds__(256) void kv8_keep(const ktir_kv8_keep_t d, int* err) {
  const ktir_kv8_t& c = d.cache;
  const int l = threadIdx.x & 63, hv = (int)blockIdx.y * 4 + uni((int)(threadIdx.x >> 6));
  if (hv >= 2 * c.heads) return;
  const int64_t head = hv >> 1, s = blockIdx.x;
  const bool is_v = hv & 1;
  const Seq q = seq_of(d.batch, c.page, s, err);
  const KTIR_G(int32_t)*path = ints(d.path) + s * d.path_row, *table = ints(d.batch.table) + s * d.batch.table_row;
  const int before = uni(q.n_kv - q.n_new), shift = __builtin_ctz((uint32_t)c.page), rows = (int)c.page;
  int n = ints(d.kept)[s];
  if (n < 0 || n > d.depth || n > q.n_new) {
    *err = OUT_OF_RANGE;
    n = n < 0 ? 0 : n > d.depth ? (int)d.depth : n;
  }
  if (before < 0) {
    if (n > 0) *err = OUT_OF_RANGE;
    return;
  }
  // the first entry that is none, and the first that moves
  int good = n, from = n;
  for (int base = 0; base < n; base += 64) {
    const int i = base + l;
    bool bad = false, moves = false;
    if (i < n) {
      const int p = path[i], last = i ? path[i - 1] : -1;
      bad = p <= last || p >= q.n_new || before + p >= q.n_held;
      moves = p != i;
      if (!bad) {
        const int a = table[(before + i) >> shift], b = table[(before + p) >> shift];
        bad = (uint32_t)a >= (uint64_t)c.pages || (uint32_t)b >= (uint64_t)c.pages;
      }
    }
    const uint64_t stop = __ballot(bad), go = __ballot(moves);
    if (from == n && go) from = base + __builtin_ctzll(go);
    if (stop) {
      good = base + __builtin_ctzll(stop);
      *err = OUT_OF_RANGE;
      break;
    }
  }
  n = uni(good);
  from = uni(from);
  if (from >= n) return;

  const uint64_t codes = is_v ? c.v + head * c.v_head : c.k + head * c.k_head, scales = is_v ? c.v_scale + head * c.vs_head * 4 : c.k_scale + head * c.ks_head * 4;
  const int64_t code_page = is_v ? c.v_page : c.k_page, tok = is_v ? c.v_tok : c.k_tok, scale_page = is_v ? c.vs_page : c.ks_page;
  auto scale_of = [&](int64_t page) { return (KTIR_G(float)*)scales + page * scale_page; };
  auto row_at = [&](int64_t page, int row) { return (KTIR_G(uint8_t)*)codes + page * code_page + row * tok; };
  const int G = (int)c.columns >> 4, per = 64 / G, r = l / G, col = (l - r * G) * 16;
  const bool mine = r < per;

  for (int p = (before + from) >> shift; p <= (before + n - 1) >> shift; ++p) {
    const int first = p << shift, lo = first > before ? first - before : 0;              // the path's entries of this page: from lo
    const int hi = (int64_t)first + rows - before < n ? first - before + rows : n;       // to hi
    const int64_t page = table[p];
    // entries of other pages: the largest value; whether something stays
    float top = 0.f;
    bool finite = true, stays = first < before;
    int came = 0;
    for (int i = lo; i < hi; i += per) {
      const int at = i + r;
      if (!mine || at >= hi) continue;
      const int src = before + path[at];
      if (src >> shift == p) {
        stays = true;
        continue;
      }
      came = 1;
      const int64_t sp = table[src >> shift];
      const float sc = *scale_of(sp);
      finite = finite && sc < __builtin_inff();
      const u4_t w = *(const KTIR_G(u4_t)*)(row_at(sp, src & (rows - 1)) + col);
      float most = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float x[4];
        values4<CODE>(w[k], x);
#pragma unroll
        for (int y = 0; y < 4; ++y) most = __builtin_fmaxf(most, __builtin_fabsf(x[y]));
      }
      top = __builtin_fmaxf(top, most * sc);
    }
    for (int o = 32; o; o >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o));
    finite = __all(finite);
    stays = __any(stays);
    came = __any(came);
    const float scale = *scale_of(page);
    float now = scale;
    if (came) {
      now = __builtin_fmaxf(top * PER_TOP<CODE>, LEAST_SCALE);
      if (stays && !(now >= scale)) now = scale;            // a page that was NaN stays so
      if (!finite) now = __builtin_nanf("");
    }
    const bool nan = !(now < __builtin_inff()), grown = came && stays && now > scale;
    const float inv = 1.f / now, again = scale * inv;
    auto rounded = [&](u4_t w, float ratio) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float x[4];
        values4<CODE>(w[k], x);
#pragma unroll
        for (int y = 0; y < 4; ++y) x[y] *= ratio;
        w[k] = codes4<CODE, CODE == KTIR_E4M3>(x);
      }
      return w;
    };
    if (grown)
      for (int row = r; mine && row < before - first; row += per) {
        KTIR_G(u4_t)* w = (KTIR_G(u4_t)*)(row_at(page, row) + col);
        *w = rounded(*w, again);
      }
    for (int i = lo; i < hi; i += per) {
      const int at = i + r;
      const bool on = mine && at < hi;
      const int src = before + (on ? path[at] : 0), row = (before + at) & (rows - 1);
      const bool here = src >> shift == p;
      const int64_t sp = table[src >> shift];
      u4_t w = {0, 0, 0, 0};
      if (on) w = *(const KTIR_G(u4_t)*)(row_at(sp, src & (rows - 1)) + col);
      if (!here) w = nan ? u4_t{0, 0, 0, 0} : rounded(w, *scale_of(sp) * inv);
      else if (grown) w = rounded(w, again);
      // (a lane's place may be another's source: no lane stores before all have loaded)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (on) *(KTIR_G(u4_t)*)(row_at(page, row) + col) = w;
    }
    if (came && l == 0) *scale_of(page) = now;
  }
}

}  // namespace ktir

using namespace ktir;

extern "C" int ktir_launch_draft_tree(const ktir_draft_tree_t* d) {
  constexpr const char* ME = "ktir_launch_draft_tree";
  if (!d) return set_error(KTIR_E_ARG, "%s: no descriptor", ME);
  if (d->seqs < 0 || d->seqs > (1 << 24) || d->tokens < 0 || d->tokens > INT32_MAX)
    return set_error(KTIR_E_ARG, "%s: %lld sequences, %lld tokens", ME, (long long)d->seqs, (long long)d->tokens);
  if (d->words < 1 || d->words > TREE_WORDS)
    return set_error(KTIR_E_UNSUPPORTED, "%s: masks of %lld words (1 to %lld)", ME, (long long)d->words, (long long)TREE_WORDS);
  if (d->window < 0 || d->window > INT32_MAX) return set_error(KTIR_E_ARG, "%s: window %lld", ME, (long long)d->window);
  if (d->seqs == 0 || d->tokens == 0) return KTIR_OK;
  if (!d->parents || !d->q_start || !d->kv_len || !d->mask || !d->positions || ((d->parents | d->q_start | d->kv_len | d->mask | d->positions) & 3))
    return set_error(KTIR_E_ARG, "%s: an array is missing or off 4-byte bounds", ME);
  if (d->mask_row < 0 || d->mask_row > ((int64_t)1 << 40) || (d->tokens > 1 && d->mask_row < d->words))
    return set_error(KTIR_E_ARG, "%s: rows of the mask overlap (stride %lld)", ME, (long long)d->mask_row);
  const Strided mask(d->mask, d->words * 4, d->tokens, d->mask_row * 4), positions(d->positions, d->tokens * 4);
  const Strided in[3] = {{d->parents, d->tokens * 4}, {d->q_start, (d->seqs + 1) * 4}, {d->kv_len, d->seqs * 4}};
  bool good = apart(mask, positions);
  for (const Strided& x : in) good = good && apart(mask, x) && apart(positions, x);
  if (!good) return set_error(KTIR_E_ARG, "%s: an output overlaps another array", ME);
  const int rc = ready(ME);
  if (rc != KTIR_OK) return rc;
  OnDevice on;
  if (!on.ok()) return set_error(KTIR_E_HIP, "%s: no device", ME);
  hipLaunchKernelGGL(draft_tree, dim3((unsigned)d->seqs, (unsigned)((d->words + 7) / 8)), dim3(256), 0, stream_of(d->stream), *d, device_error_flag());
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}

extern "C" int ktir_launch_kv8_keep(const ktir_kv8_keep_t* d) {
  constexpr const char* ME = "ktir_launch_kv8_keep";
  if (!d) return set_error(KTIR_E_ARG, "%s: no descriptor", ME);
  int rc = check_kv8(ME, d->cache, true);
  if (rc == KTIR_OK) rc = check_batch(ME, d->batch, d->cache);
  if (rc != KTIR_OK) return rc;
  if (d->depth < 0 || d->depth > INT32_MAX || d->path_row < 0 || d->path_row > ((int64_t)1 << 40))
    return set_error(KTIR_E_ARG, "%s: paths of %lld tokens, stride %lld", ME, (long long)d->depth, (long long)d->path_row);
  if (d->batch.seqs == 0 || d->batch.tokens == 0 || d->depth == 0) return KTIR_OK;
  if (!d->path || !d->kept || ((d->path | d->kept) & 3)) return set_error(KTIR_E_ARG, "%s: paths missing or off 4-byte bounds", ME);
  const BatchParts batch(d->batch);
  const Strided path(d->path, d->depth * 4, d->batch.seqs, d->path_row * 4), kept(d->kept, d->batch.seqs * 4);
  for (const Strided& out : CacheParts(d->cache).x)
    if (!batch.clear_of(out) || !apart(out, path) || !apart(out, kept))
      return set_error(KTIR_E_ARG, "%s: the cache overlaps the table, offsets, lengths or paths", ME);
  rc = ready(ME);
  if (rc != KTIR_OK) return rc;
  OnDevice on;
  if (!on.ok()) return set_error(KTIR_E_HIP, "%s: no device", ME);
  const dim3 grid((unsigned)d->batch.seqs, (unsigned)((2 * d->cache.heads + 3) / 4));
  if (grid.y > 65535) return set_error(KTIR_E_UNSUPPORTED, "%s: %lld heads in one launch", ME, (long long)d->cache.heads);
  const hipStream_t st = stream_of(d->stream);
  if (d->cache.dtype == KTIR_I8) hipLaunchKernelGGL(kv8_keep<KTIR_I8>, grid, dim3(256), 0, st, *d, device_error_flag());
  else hipLaunchKernelGGL(kv8_keep<KTIR_E4M3>, grid, dim3(256), 0, st, *d, device_error_flag());
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}
