// The key / value cache in 8 bits: checks of its descriptors, and the append of
// new tokens with a scale for each page and head.
//
// Append.  Bound: bytes, 2 a value in and 1 out, and the chain offsets -> table and
// values -> scale for few tokens.  A page's part of a head is the work of one group of
// wavefronts, so its maximum needs no atomics and its older rows no lock.  Measured:
// 8192 tokens of 8 heads of 128, K and V, 50 MB, 12.4 us = 4.1 TB/s (63 us with the values
// read twice, an element a thread); 64 tokens of as many sequences 4.3 us, a launch.
#include "ktir_kv8_codes.h"

namespace ktir {

int ready(const char* what) {
  if (device() < 0 || !device_error_flag()) return set_error(KTIR_E_ARG, "%s: ktir_init has not run", what);
  return KTIR_OK;
}

int check_rows3(const char* what, const ktir_rows3_t& r, int64_t tokens, int64_t heads, int64_t columns, bool written) {
  if (!r.ptr) return set_error(KTIR_E_ARG, "%s: a tensor is missing", what);
  constexpr int64_t FAR = (int64_t)1 << 40;
  if (r.tok < 0 || r.head < 0 || r.tok > FAR || r.head > FAR) return set_error(KTIR_E_ARG, "%s: strides %lld, %lld", what, (long long)r.tok, (long long)r.head);
  if (!written) return KTIR_OK;
  // rows of an output must not overlap: in order of their strides each dimension steps over the smaller one
  int64_t n[2] = {heads, tokens}, st[2] = {r.head, r.tok};
  if (st[0] > st[1]) {
    n[0] = tokens, n[1] = heads;
    st[0] = r.tok, st[1] = r.head;
  }
  int64_t span = columns;
  for (int i = 0; i < 2; ++i) {
    if (n[i] <= 1) continue;
    if (st[i] < span) return set_error(KTIR_E_ARG, "%s: rows of an output overlap (strides %lld, %lld)", what, (long long)r.tok, (long long)r.head);
    span += (n[i] - 1) * st[i];
  }
  return KTIR_OK;
}

bool same(const Strided& a, const Strided& b) {
  bool good = a.ptr == b.ptr && a.width == b.width;
  for (int i = 0; i < 3; ++i) good = good && a.count[i] == b.count[i] && (a.count[i] == 1 || a.step[i] == b.step[i]);
  return good;
}

// Whether `off` + sum_i d_i step_i lies between lo and hi for some d_i of first_i to
// last_i; steps in falling order, so that few d_i can do (the rows of an output do not
// overlap: a step is no less than the reach of those after it).
static bool reaches(int64_t off, int64_t lo, int64_t hi, int dims, const int64_t* step, const int64_t* first, const int64_t* last) {
  if (dims == 0) return lo <= off && off <= hi;
  int64_t down = 0, up = 0;
  for (int i = 1; i < dims; ++i) down += first[i] * step[i], up += last[i] * step[i];
  auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
  int64_t d = -floor_div(off + up - lo, *step), most = floor_div(hi - off - down, *step);
  if (d < *first) d = *first;
  if (most > *last) most = *last;
  for (; d <= most; ++d)
    if (reaches(off + d * *step, lo, hi, dims - 1, step + 1, first + 1, last + 1)) return true;
  return false;
}

// Dimensions that both step alike are followed (parts of one projection, K and V of one
// allocation, scales behind the codes of their page); in others a tensor counts as
// all that lies between its first and last byte.
bool apart_within(Strided a, Strided b) {
  int dims = 0;
  int64_t step[3], first[3], last[3];
  for (int i = 0; i < 3; ++i) {
    if (a.count[i] > 1 && b.count[i] > 1 && a.step[i] != b.step[i]) {
      for (Strided* x : {&a, &b}) x->width += (x->count[i] - 1) * x->step[i], x->count[i] = 1;
      continue;
    }
    const int64_t s = a.count[i] > 1 ? a.step[i] : b.step[i];
    if (s == 0 || (a.count[i] == 1 && b.count[i] == 1)) continue;
    int at = dims++;
    for (; at > 0 && step[at - 1] < s; --at) step[at] = step[at - 1], first[at] = first[at - 1], last[at] = last[at - 1];
    step[at] = s, first[at] = 1 - a.count[i], last[at] = b.count[i] - 1;
  }
  return !reaches((int64_t)(b.ptr - a.ptr), 1 - b.width, a.width - 1, dims, step, first, last);
}

static int check_codes(const char* what, uint64_t ptr, int64_t page, int64_t tok, int64_t head, const ktir_kv8_t& c, bool written) {
  constexpr int64_t FAR = (int64_t)1 << 40;
  if (!ptr) return set_error(KTIR_E_ARG, "%s: a cache is missing", what);
  if (page < 0 || tok < 0 || head < 0 || page > FAR || tok > FAR || head > FAR)
    return set_error(KTIR_E_ARG, "%s: cache strides %lld, %lld, %lld", what, (long long)page, (long long)tok, (long long)head);
  if (tok > (1 << 22)) return set_error(KTIR_E_UNSUPPORTED, "%s: tokens of a page lie %lld bytes apart", what, (long long)tok);
  if ((ptr | page | tok | head) & 15) return set_error(KTIR_E_UNSUPPORTED, "%s: cache rows lie off 16-byte bounds", what);
  if (!written) return KTIR_OK;
  int64_t n[3] = {c.pages, c.page, c.heads}, st[3] = {page, tok, head};
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2 - i; ++j)
      if (st[j] > st[j + 1]) {
        int64_t x = st[j];
        st[j] = st[j + 1], st[j + 1] = x;
        x = n[j], n[j] = n[j + 1], n[j + 1] = x;
      }
  int64_t span = c.columns;
  for (int i = 0; i < 3; ++i) {
    if (n[i] <= 1) continue;
    if (st[i] < span) return set_error(KTIR_E_ARG, "%s: rows of the cache overlap", what);
    span += (n[i] - 1) * st[i];
  }
  return KTIR_OK;
}

int check_kv8(const char* what, const ktir_kv8_t& c, bool written) {
  if (c.pages < 1 || c.heads < 1 || c.pages > INT32_MAX || c.heads > 65536)
    return set_error(KTIR_E_ARG, "%s: a cache of %lld pages and %lld heads", what, (long long)c.pages, (long long)c.heads);
  if (c.page < 16 || c.page > 256 || (c.page & (c.page - 1)))
    return set_error(KTIR_E_UNSUPPORTED, "%s: pages of %lld tokens (a power of two from 16 to 256)", what, (long long)c.page);
  if (c.columns < 16 || c.columns > 256 || (c.columns & 15))
    return set_error(KTIR_E_UNSUPPORTED, "%s: heads of %lld columns (a multiple of 16 up to 256)", what, (long long)c.columns);
  if (c.dtype != KTIR_I8 && c.dtype != KTIR_E4M3) return set_error(KTIR_E_UNSUPPORTED, "%s: codes of dtype %d", what, c.dtype);
  int rc = check_codes(what, c.k, c.k_page, c.k_tok, c.k_head, c, written);
  if (rc == KTIR_OK) rc = check_codes(what, c.v, c.v_page, c.v_tok, c.v_head, c, written);
  if (rc != KTIR_OK) return rc;
  constexpr int64_t FAR = (int64_t)1 << 40;
  const int64_t st[4] = {c.ks_page, c.ks_head, c.vs_page, c.vs_head};
  for (int64_t x : st)
    if (x < 0 || x > FAR) return set_error(KTIR_E_ARG, "%s: stride %lld of the scales", what, (long long)x);
  if (!c.k_scale || !c.v_scale || ((c.k_scale | c.v_scale) & 3)) return set_error(KTIR_E_ARG, "%s: scales missing or off 4-byte bounds", what);
  if (written && ((c.pages > 1 && (!c.ks_page || !c.vs_page)) || (c.heads > 1 && (!c.ks_head || !c.vs_head))))
    return set_error(KTIR_E_ARG, "%s: pages or heads share a scale", what);
  if (!written) return KTIR_OK;
  const CacheParts parts(c);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < i; ++j)
      if (!apart(parts.x[i], parts.x[j])) return set_error(KTIR_E_ARG, "%s: the caches or scales of keys and values overlap", what);
  return KTIR_OK;
}

int check_batch(const char* what, const ktir_kv8_batch_t& b, const ktir_kv8_t& c) {
  if (b.seqs < 0 || b.seqs > (1 << 24) || b.tokens < 0 || b.tokens > INT32_MAX || b.width < 0 || b.width > INT32_MAX)
    return set_error(KTIR_E_ARG, "%s: %lld sequences, %lld tokens, tables of %lld pages", what, (long long)b.seqs, (long long)b.tokens,
                     (long long)b.width);
  if (b.seqs == 0 || b.tokens == 0) return KTIR_OK;
  if (!b.q_start || !b.kv_len || (!b.table && b.width) || ((b.q_start | b.kv_len | b.table) & 3))
    return set_error(KTIR_E_ARG, "%s: table, offsets or lengths missing or off 4-byte bounds", what);
  if (b.table_row < 0 || b.table_row > ((int64_t)1 << 40)) return set_error(KTIR_E_ARG, "%s: table stride %lld", what, (long long)b.table_row);
  return KTIR_OK;
}

// ---- append ----------------------------------------------------------------

constexpr int APPEND_KEPT = 4;       // units of 16 values that a thread keeps between the two passes

// W wavefronts (1 or 4) per page that new tokens fall in, head, and K or V: a thread
// takes units of 16 columns of a row.  The new values are read once, into
// registers, up to 64 W APPEND_KEPT units; units past those (pages of 256 rows of 256
// columns) are read again, from the cache.
template <int CODE, bool BF16, int W>
__global__ __launch_bounds__(256) void kv8_append(const ktir_kv8_append_t d, int* err) {
  __shared__ uint32_t tops[4];
  const ktir_kv8_t& c = d.cache;
  const int wave = uni((int)(threadIdx.x >> 6)), tid = W == 1 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
  const int hv = W == 1 ? (int)blockIdx.y * 4 + wave : (int)blockIdx.y;
  if (hv >= 2 * c.heads) return;
  const int64_t head = hv >> 1;
  const bool is_v = hv & 1;
  int64_t s, nth;
  const int shift = __builtin_ctz((uint32_t)c.page);
  const Seq q = seq_of_slot(d.batch, c.page, 1, shift, 2, blockIdx.x, &s, &nth, err);
  if (nth < 0) return;
  const int64_t pos0 = (int64_t)q.n_kv - q.n_new, from = pos0 < 0 ? 0 : pos0;      // the first position that is stored
  const int64_t p = (from >> shift) + nth;                                       // the page's number in the sequence
  const int64_t lo = p << shift < from ? from : p << shift, hi = (p + 1) << shift < q.n_held ? (p + 1) << shift : q.n_held;
  if (lo >= hi) return;
  const int64_t at = ints(d.batch.table)[s * d.batch.table_row + p];

  const ktir_rows3_t& in = is_v ? d.v : d.k;
  const int G = (int)c.columns >> 4, per = 64 * W / G, r = tid / G, col = (tid - r * G) * 16;     // rows a pass; this thread's
  const int n = (int)(hi - lo), r0 = (int)(lo & (c.page - 1));
  const bool wide = !((in.ptr | (uint64_t)in.tok * 2 | (uint64_t)in.head * 2) & 15), mine = r < per;
  const int64_t e0 = (q.start + lo - pos0) * in.tok + head * in.head + col;
  New16 x[APPEND_KEPT];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < APPEND_KEPT; ++i)
    if (mine && i * per + r < n) x[i] = new16(in.ptr, e0 + (i * per + r) * in.tok, wide);
#pragma unroll
  for (int i = 0; i < APPEND_KEPT; ++i)
    if (mine && i * per + r < n) top = top16(x[i], top);
  for (int row = APPEND_KEPT * per + r; mine && row < n; row += per) top = top16(new16(in.ptr, e0 + row * in.tok, wide), top);
  if (at < 0 || at >= c.pages) {
    *err = OUT_OF_RANGE;
    return;
  }
  KTIR_G(uint8_t)* codes = (KTIR_G(uint8_t)*)(is_v ? c.v + at * c.v_page + head * c.v_head : c.k + at * c.k_page + head * c.k_head) + col;
  const int tok = (int)(is_v ? c.v_tok : c.k_tok);
  KTIR_G(float)* scale = is_v ? (KTIR_G(float)*)c.v_scale + at * c.vs_page + head * c.vs_head
                              : (KTIR_G(float)*)c.k_scale + at * c.ks_page + head * c.ks_head;
  const float before = r0 ? *scale : 0.f;
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const uint32_t y = __shfl_xor(top, o);
    top = top > y ? top : y;
  }
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) tops[wave] = top;
    __syncthreads();                       // also: every wavefront has read the scale before it changes
#pragma unroll
    for (int i = 0; i < W; ++i) top = top > tops[i] ? top : tops[i];
  }
  const float most = BF16 ? __uint_as_float(top << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)top);
  float now = __builtin_fmaxf(most * PER_TOP<CODE>, LEAST_SCALE);
  if (!(now >= before)) now = before;                     // a page that was NaN stays so
  if (!(most < __builtin_inff())) now = __builtin_nanf("");
  const bool nan = !(now < __builtin_inff());
  const float inv = 1.f / now;
  if (now > before && mine) {              // older rows rounded to the new scale
    const float ratio = before * inv;
    for (int row = r; row < r0; row += per) {
      KTIR_G(u4_t)* w = (KTIR_G(u4_t)*)(codes + row * tok);
      u4_t y = *w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v[4];
        values4<CODE>(y[i], v);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] *= ratio;
        y[i] = codes4<CODE, CODE == KTIR_E4M3>(v);
      }
      *w = y;
    }
  }
  const u4_t none = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < APPEND_KEPT; ++i)
    if (mine && i * per + r < n) *(KTIR_G(u4_t)*)(codes + (r0 + i * per + r) * tok) = nan ? none : codes16<BF16>(x[i], inv, CODE);
  for (int row = APPEND_KEPT * per + r; mine && row < n; row += per)
    *(KTIR_G(u4_t)*)(codes + (r0 + row) * tok) = nan ? none : codes16<BF16>(new16(in.ptr, e0 + row * in.tok, wide), inv, CODE);
  if (tid == 0) *scale = now;
}

template <int CODE, bool BF16>
static void append_go(const ktir_kv8_append_t& d, int64_t slots, hipStream_t st) {
  // a page's units fit into one wavefront's registers: four pages or heads share a workgroup
  const int64_t hv = 2 * d.cache.heads;
  if (d.cache.page * (d.cache.columns / 16) <= 64 * APPEND_KEPT)
    hipLaunchKernelGGL((kv8_append<CODE, BF16, 1>), dim3((unsigned)slots, (unsigned)((hv + 3) / 4)), dim3(256), 0, st, d, device_error_flag());
  else
    hipLaunchKernelGGL((kv8_append<CODE, BF16, 4>), dim3((unsigned)slots, (unsigned)hv), dim3(256), 0, st, d, device_error_flag());
}

}  // namespace ktir

using namespace ktir;

extern "C" int ktir_launch_kv8_append(const ktir_kv8_append_t* d) {
  constexpr const char* ME = "ktir_launch_kv8_append";
  if (!d) return set_error(KTIR_E_ARG, "%s: no descriptor", ME);
  if (d->dtype != KTIR_F16 && d->dtype != KTIR_BF16) return set_error(KTIR_E_UNSUPPORTED, "%s: dtype %d", ME, d->dtype);
  int rc = check_kv8(ME, d->cache, true);
  if (rc == KTIR_OK) rc = check_batch(ME, d->batch, d->cache);
  if (rc != KTIR_OK || d->batch.seqs == 0 || d->batch.tokens == 0) return rc;
  rc = check_rows3(ME, d->k, d->batch.tokens, d->cache.heads, d->cache.columns, false);
  if (rc == KTIR_OK) rc = check_rows3(ME, d->v, d->batch.tokens, d->cache.heads, d->cache.columns, false);
  if (rc != KTIR_OK) return rc;
  const BatchParts batch(d->batch);
  const Strided k = rows_of(d->k, d->batch.tokens, d->cache.heads, d->cache.columns, 2), v = rows_of(d->v, d->batch.tokens, d->cache.heads, d->cache.columns, 2);
  for (const Strided& out : CacheParts(d->cache).x) {
    if (!apart(out, k) || !apart(out, v)) return set_error(KTIR_E_ARG, "%s: the cache overlaps the new keys or values", ME);
    if (!batch.clear_of(out)) return set_error(KTIR_E_ARG, "%s: the cache overlaps the table, offsets or lengths", ME);
  }
  rc = ready(ME);
  if (rc != KTIR_OK) return rc;
  OnDevice on;
  if (!on.ok()) return set_error(KTIR_E_HIP, "%s: no device", ME);
  // a sequence's n new tokens touch at most floor(n / page) + 2 pages
  const int64_t slots = d->batch.tokens / d->cache.page + 2 * d->batch.seqs;
  if (slots > INT32_MAX || d->cache.heads > 32767) return set_error(KTIR_E_UNSUPPORTED, "%s: %lld pages, %lld heads in one launch", ME, (long long)slots, (long long)d->cache.heads);
  const hipStream_t st = stream_of(d->stream);
  if (d->cache.dtype == KTIR_I8) d->dtype == KTIR_BF16 ? append_go<KTIR_I8, true>(*d, slots, st) : append_go<KTIR_I8, false>(*d, slots, st);
  else d->dtype == KTIR_BF16 ? append_go<KTIR_E4M3, true>(*d, slots, st) : append_go<KTIR_E4M3, false>(*d, slots, st);
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}
