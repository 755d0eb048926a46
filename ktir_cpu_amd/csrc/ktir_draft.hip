// Drafted tokens: positions and ancestor masks of a tree, and the accepted path's
// entries of the 8-bit cache.
#include "ktir_kv8_codes.h"

namespace ktir {

constexpr int64_t TREE_WORDS = 32;           // of a token's mask

// ---- the tree ----------------------------------------------------------------
//
// Tokens come after their parents, so 32 of them (a word of the masks) have all other ancestors among
// the tokens before.  One thread a token: first up the line within its word, which half a wavefront holds, in 5
// doublings; where that leaves the word, the row of the ancestor it comes to has the other words, which are copied word
// by word of the sequence.  Bound: latency, the chain offsets -> parents, then a step of LDS and a barrier for each word.
// 64 sequences of up to 64 tokens 3.8 to 4.1 us (2.7 in a graph), 24 of up to 500, with a window, 6.8; 10.7 with the line walked token
// by token and the window's bits dropped one by one, 41 without the words.  Threads for 4, 16 or 32 words: in a graph
// 512 sequences of up to 64 tokens take 2.9, 3.7 and 6.8 us, of up to 500 8.1 with 16 words and 13.8 with 32.

template <int WORDS>
__global__ __launch_bounds__(32 * WORDS) void draft_tree(const ktir_draft_tree_t d, int* err) {
  constexpr int N = 32 * WORDS, PITCH = WORDS + 1;
  __shared__ uint32_t rows[N * PITCH];
  __shared__ int line[N], depths[N];                // the first ancestor before a token's word; how many ancestors
  const int i = threadIdx.x, word = i >> 5;
  const int64_t s = blockIdx.x;
  const int64_t a = ints(d.q_start)[s], e = ints(d.q_start)[s + 1];
  const int kv = ints(d.kv_len)[s];
  const int64_t start = a < 0 ? 0 : a < d.tokens ? a : d.tokens, end = e < start ? start : e < d.tokens ? e : d.tokens;
  if (start != a || end != e || kv < 0 || end - start > 32 * d.words) {
    *err = OUT_OF_RANGE;
    if (end - start > 32 * d.words) return;
  }
  const int n = (int)(end - start);                 // N at most
  int p = -1;
  if (i < n) {
    p = ints(d.parents)[start + i];
    if (p < -1 || p >= i) *err = OUT_OF_RANGE, p = -1;
  }
  uint32_t bits = 1u << (i & 31);
#pragma unroll
  for (int o = 0; o < 5; ++o) {                     // (a word is half a wavefront)
    const bool inside = p >= word * 32;
    const int at = inside ? p & 31 : i & 31, up = __shfl(p, at, 32);
    bits |= __shfl(bits, at, 32);
    p = inside ? up : p;
  }
  const int steps = __builtin_popcount(bits) - 1;
  for (int w = word; w < WORDS; ++w) rows[i * PITCH + w] = w == word ? bits : 0u;
  line[i] = p;
  if (p < 0) depths[i] = steps;
  __syncthreads();
  int ups[WORDS];
#pragma unroll
  for (int b = 0; b < WORDS; ++b) ups[b] = line[32 * b + (i & 31)];
#pragma unroll
  for (int b = 0; b < WORDS; ++b) {                 // one thread a word of a row, and one a row for its depth
    if (32 * b >= n) break;
    const int t = 32 * b + (i & 31), w = i >> 5, up = ups[b];
    if (w < b) rows[t * PITCH + w] = up < 0 ? 0u : rows[up * PITCH + w];
    if (word == b && p >= 0) depths[i] = steps + 1 + depths[p];
    __syncthreads();
  }
  if (i < n) ((KTIR_G(int32_t)*)d.positions)[start + i] = (kv < 0 ? 0 : kv) - n + depths[i];
  if (d.window) {                                   // the highest `window` bits of each row
    if (i < n && depths[i] >= d.window) {
      int left = (int)d.window;
      uint32_t y[WORDS];
#pragma unroll
      for (int w = 0; w < WORDS; ++w) y[w] = rows[i * PITCH + w];
#pragma unroll
      for (int w = WORDS - 1; w >= 0; --w) {
        const int some = __builtin_popcount(y[w]);
        if (left < some) {                          // the highest `left` of a word's: from the bit on below which it has one more
          int low = 0;
#pragma unroll
          for (int o = 16; o; o >>= 1) low += __builtin_popcount(y[w] >> (low + o)) > left ? o : 0;
          y[w] = left ? y[w] & ~1u << low : 0u;
        }
        left = left > some ? left - some : 0;
      }
#pragma unroll
      for (int w = 0; w < WORDS; ++w) rows[i * PITCH + w] = y[w];
    }
    __syncthreads();
  }
  const int words = (int)d.words, each = N / words, w = i % words;
  if (i < each * words)
    for (int t = i / words; t < n; t += each) ((KTIR_G(uint32_t)*)d.mask)[(start + t) * d.mask_row + w] = rows[t * PITCH + w];
}

// ---- the kept path -----------------------------------------------------------
//
// One wavefront for a sequence, a KV head, and K or V.  Entries only move down and in order, so what a
// page gets is read before its place is written: pages in order, and in a page the rows of
// one pass of the wavefront (64 units of 16 columns), all read, then written.  Bound: latency, offsets and path ->
// table -> scales and codes, for each page; a lane has the place, page and scale that one entry of 64 comes from.  One sequence of
// 16 drafts 4.3 us, which is the launch, 256 of up to 64 10.2 (12.7 with each entry's place looked up by every lane).

constexpr int KEEP_KEPT = 2;         // passes of rows that stay in registers between the maximum and the codes

template <int CODE>
__global__ __launch_bounds__(256) void kv8_keep(const ktir_kv8_keep_t d, int* err) {
  const ktir_kv8_t& c = d.cache;
  const int l = threadIdx.x & 63, hv = (int)blockIdx.y * 4 + uni((int)(threadIdx.x >> 6));
  if (hv >= 2 * c.heads) return;
  const int64_t head = hv >> 1, s = blockIdx.x;
  const bool is_v = hv & 1;
  const KTIR_G(int32_t)*path = ints(d.path) + s * d.path_row, *table = ints(d.batch.table) + s * d.batch.table_row;
  // (the first entries and their count on their way with the offsets)
  int mine = l < d.depth ? path[l] : 0, n = ints(d.kept)[s];
  const Seq q = seq_of(d.batch, c.page, s, err);
  const int before = uni(q.n_kv - q.n_new), held = uni(q.n_held), fresh = uni(q.n_new), shift = __builtin_ctz((uint32_t)c.page), rows = (int)c.page;
  n = uni(n);
  if (n < 0 || n > d.depth || n > fresh) {
    *err = OUT_OF_RANGE;
    n = n < 0 ? 0 : n > d.depth ? (int)d.depth : n;
  }
  if (before < 0) {
    if (n > 0) *err = OUT_OF_RANGE;
    return;
  }
  const uint64_t codes = is_v ? c.v + head * c.v_head : c.k + head * c.k_head, scales = is_v ? c.v_scale + head * c.vs_head * 4 : c.k_scale + head * c.ks_head * 4;
  const int64_t code_page = is_v ? c.v_page : c.k_page, tok = is_v ? c.v_tok : c.k_tok, scale_page = is_v ? c.vs_page : c.ks_page;
  auto scale_of = [&](int64_t page) { return (KTIR_G(float)*)scales + page * scale_page; };
  auto row_at = [&](int64_t page, int row) { return (KTIR_G(uint8_t)*)codes + page * code_page + row * tok; };

  // entries base .. base + 63, one a lane: the place in the cache that each comes from, its page and scale, and its new page
  int base = 0, src = 0, from_page = 0, to_page = 0;
  float from_scale = 0.f;
  // the first entry that is none, and the first that moves
  int good = n, from = n;
  for (base = 0; base < n; base += 64) {
    const int i = base + l;
    if (base) mine = i < n ? path[i] : 0;
    int last = __shfl_up(mine, 1);
    if (l == 0) last = base ? path[base - 1] : -1;
    src = before + mine;
    bool bad = i < n && (mine <= last || mine >= fresh || src >= held);
    if (i < n && !bad) {
      to_page = table[(before + i) >> shift];
      from_page = table[src >> shift];
      bad = (uint32_t)to_page >= (uint64_t)c.pages || (uint32_t)from_page >= (uint64_t)c.pages;
    }
    const uint64_t stop = __ballot(bad), go = __ballot(i < n && mine != i);
    if (from == n && go) from = base + __builtin_ctzll(go);
    if (stop) {
      good = base + __builtin_ctzll(stop);
      *err = OUT_OF_RANGE;
      break;
    }
    if (n <= 64) break;
  }
  n = good;
  if (from >= n) return;
  if (base + l < n) from_scale = *scale_of(from_page);
  auto fetch = [&](int at) {                 // entries from `at` on, where the ones at hand are others
    base = at;
    if (at + l >= n) return;
    src = before + path[at + l];
    to_page = table[(before + at + l) >> shift];
    from_page = table[src >> shift];
    from_scale = *scale_of(from_page);
  };
  const int G = (int)c.columns >> 4, per = 64 / G, r = l / G, col = (l - r * G) * 16;
  auto need = [&](int at, int end) {         // entries [at, end), 64 at most, at hand
    if (at < base || end > base + 64) fetch(at);
  };
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

  for (int p = (before + from) >> shift; p <= (before + n - 1) >> shift; ++p) {
    const int first = p << shift, lo = first > before ? first - before : 0;              // the path's entries of this page: from lo
    const int hi = (int64_t)first + rows - before < n ? first - before + rows : n;       // to hi
    // a unit of each row: where it comes from, whether from this page, its scale and codes
    struct Unit {
      int64_t page;
      float scale;
      bool on, here;
      u4_t w;
    };
    auto load = [&](int i, Unit& u) {
      need(i, i + per < hi ? i + per : hi);
      const int k = i + r - base;
      u.on = r < per && i + r < hi;
      const int place = __shfl(src, k & 63);
      u.page = __shfl(from_page, k & 63);
      u.scale = __shfl(from_scale, k & 63);
      u.here = place >> shift == p;
      u.w = u4_t{0, 0, 0, 0};
      if (u.on) u.w = *(const KTIR_G(u4_t)*)(row_at(u.page, place & (rows - 1)) + col);
    };
    need(lo, lo + 64 < hi ? lo + 64 : hi);
    const int64_t page = __shfl(to_page, lo - base);
    const float scale = *scale_of(page);
    // entries of other pages: the largest value; whether something stays
    float top = 0.f;
    bool finite = true, stays = first < before, came = false;
    auto look = [&](const Unit& u) {
      if (!u.on) return;
      stays = stays || u.here;
      came = came || !u.here;
      if (u.here) return;
      finite = finite && u.scale < __builtin_inff();
      float most = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float x[4];
        values4<CODE>(u.w[k], x);
#pragma unroll
        for (int y = 0; y < 4; ++y) most = __builtin_fmaxf(most, __builtin_fabsf(x[y]));
      }
      top = __builtin_fmaxf(top, most * u.scale);
    };
    Unit unit[KEEP_KEPT];
#pragma unroll
    for (int k = 0; k < KEEP_KEPT; ++k) {
      unit[k].on = false;
      if (lo + k * per < hi) load(lo + k * per, unit[k]);
    }
#pragma unroll
    for (int k = 0; k < KEEP_KEPT; ++k) look(unit[k]);
    for (int i = lo + KEEP_KEPT * per; i < hi; i += per) {
      Unit u;
      load(i, u);
      look(u);
    }
    for (int o = 32; o; o >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o));
    finite = __all(finite);
    stays = __any(stays);
    came = __any(came);
    float now = scale;
    if (came) {
      now = __builtin_fmaxf(top * PER_TOP<CODE>, LEAST_SCALE);
      if (stays && !(now >= scale)) now = scale;            // a page that was NaN stays so
      if (!finite) now = __builtin_nanf("");
    }
    const bool nan = !(now < __builtin_inff()), grown = came && stays && now > scale;
    const float inv = 1.f / now, again = scale * inv;
    if (grown)
      for (int row = r; r < per && row < before - first; row += per) {
        KTIR_G(u4_t)* w = (KTIR_G(u4_t)*)(row_at(page, row) + col);
        *w = rounded(*w, again);
      }
    auto put = [&](int i, const Unit& u) {
      u4_t w = u.w;
      if (!u.here) w = nan ? u4_t{0, 0, 0, 0} : rounded(w, u.scale * inv);
      else if (grown) w = rounded(w, again);
      // (a lane's place may be another's source: no lane stores before all have loaded)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (u.on) *(KTIR_G(u4_t)*)(row_at(page, (before + i + r) & (rows - 1)) + col) = w;
    };
#pragma unroll
    for (int k = 0; k < KEEP_KEPT; ++k)
      if (lo + k * per < hi) put(lo + k * per, unit[k]);
    for (int i = lo + KEEP_KEPT * per; i < hi; i += per) {
      Unit u;
      load(i, u);
      put(i, u);
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
  const dim3 grid((unsigned)d->seqs);
  const hipStream_t st = stream_of(d->stream);
  if (d->words <= 4) hipLaunchKernelGGL(draft_tree<4>, grid, dim3(128), 0, st, *d, device_error_flag());
  else if (d->words <= 16) hipLaunchKernelGGL(draft_tree<16>, grid, dim3(512), 0, st, *d, device_error_flag());
  else hipLaunchKernelGGL(draft_tree<32>, grid, dim3(1024), 0, st, *d, device_error_flag());
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
