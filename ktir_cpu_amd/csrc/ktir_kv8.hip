// The key / value cache in 8 bits: checks of its descriptors, and the append of
// new tokens with a scale for each page and head.
#include "ktir_serve.h"

namespace ktir {

constexpr float LEAST_SCALE = 0x1p-100f;     // codes of a page of zeros are zeros times this

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

// one code of x / scale
template <int CODE>
__device__ __forceinline__ uint8_t code_of(float x) {
  if constexpr (CODE == KTIR_I8) {
    const float r = __builtin_rintf(x);
    return (uint8_t)(int8_t)(int)__builtin_fminf(__builtin_fmaxf(r, -127.f), 127.f);
  } else {
    const float r = __builtin_fminf(__builtin_fmaxf(x, -448.f), 448.f);
    return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(r, r, 0, false) & 0xff);
  }
}

template <int CODE>
__device__ __forceinline__ float value_of(uint8_t c) {
  if constexpr (CODE == KTIR_I8) return (float)(int8_t)c;
  else return __builtin_amdgcn_cvt_f32_fp8(c, 0);
}

template <int CODE>
constexpr float TOP = CODE == KTIR_I8 ? 127.f : 448.f;

// one wavefront per page slot, head, and K or V
template <int CODE>
__global__ __launch_bounds__(64) void kv8_append_plain(const ktir_kv8_append_t d, int* err) {
  const ktir_kv8_t& c = d.cache;
  const int64_t head = blockIdx.y >> 1;
  const bool is_v = blockIdx.y & 1;
  int64_t nth;
  const int64_t s = seq_of_slot(d.batch, 1, c.page, 2, blockIdx.x, &nth);
  const Seq q = seq_of(d.batch, c.page, s, err);
  const int64_t pos0 = (int64_t)q.n_kv - q.n_new, from = pos0 < 0 ? 0 : pos0;      // the first position that is stored
  const int64_t p = from / c.page + nth;                                         // the page's number in the sequence
  const int64_t lo = p * c.page < from ? from : p * c.page, hi = (p + 1) * c.page < q.n_held ? (p + 1) * c.page : q.n_held;
  if (nth < 0 || lo >= hi) return;
  const int64_t at = ints(d.batch.table)[s * d.batch.table_row + p];
  if (at < 0 || at >= c.pages) {
    *err = OUT_OF_RANGE;
    return;
  }
  const ktir_rows3_t& in = is_v ? d.v : d.k;
  const uint64_t codes = (is_v ? c.v + at * c.v_page + head * c.v_head : c.k + at * c.k_page + head * c.k_head);
  const int64_t tok = is_v ? c.v_tok : c.k_tok;
  KTIR_G(float)* scale = is_v ? (KTIR_G(float)*)c.v_scale + at * c.vs_page + head * c.vs_head
                              : (KTIR_G(float)*)c.k_scale + at * c.ks_page + head * c.ks_head;
  const int l = threadIdx.x, n = (int)(hi - lo), r0 = (int)(lo - p * c.page), D = (int)c.columns;
  const int64_t e0 = (q.start + lo - pos0) * in.tok + head * in.head;
  float top = 0.f;
  bool bad = false;
  for (int i = l; i < n * D; i += 64) {
    const float x = __builtin_fabsf(load_elem(in.ptr, e0 + (i / D) * in.tok + i % D, d.dtype));
    bad |= !(x < __builtin_inff());
    top = __builtin_fmaxf(top, x);
  }
  for (int o = 32; o; o >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o));
  bad = __any(bad);
  const float before = r0 ? *scale : 0.f;
  float now = __builtin_fmaxf(top / TOP<CODE>, LEAST_SCALE);
  if (!(now >= before)) now = before;                     // a page that was NaN stays so
  if (bad) now = __builtin_nanf("");
  const bool nan = !(now < __builtin_inff());
  const float inv = 1.f / now;
  if (r0 && now > before) {
    const float ratio = before * inv;
    for (int i = l; i < r0 * D; i += 64) {
      KTIR_G(uint8_t)* w = (KTIR_G(uint8_t)*)codes + (i / D) * tok + i % D;
      *w = code_of<CODE>(value_of<CODE>(*w) * ratio);
    }
  }
  for (int i = l; i < n * D; i += 64) {
    const float x = load_elem(in.ptr, e0 + (i / D) * in.tok + i % D, d.dtype);
    ((KTIR_G(uint8_t)*)codes)[(r0 + i / D) * tok + i % D] = nan ? 0 : code_of<CODE>(x * inv);
  }
  if (l == 0) *scale = now;
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
  if (rc == KTIR_OK) rc = ready(ME);
  if (rc != KTIR_OK) return rc;
  OnDevice on;
  if (!on.ok()) return set_error(KTIR_E_HIP, "%s: no device", ME);
  // a sequence's n new tokens touch at most floor(n / page) + 2 pages
  const int64_t slots = d->batch.tokens / d->cache.page + 2 * d->batch.seqs;
  if (slots > INT32_MAX || d->cache.heads > 32767) return set_error(KTIR_E_UNSUPPORTED, "%s: %lld pages, %lld heads in one launch", ME, (long long)slots, (long long)d->cache.heads);
  const dim3 grid((unsigned)slots, (unsigned)(2 * d->cache.heads));
  if (d->cache.dtype == KTIR_I8) hipLaunchKernelGGL(kv8_append_plain<KTIR_I8>, grid, dim3(64), 0, stream_of(d->stream), *d, device_error_flag());
  else hipLaunchKernelGGL(kv8_append_plain<KTIR_E4M3>, grid, dim3(64), 0, stream_of(d->stream), *d, device_error_flag());
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}
