// Attention of drafted tokens over the 8-bit cache: the entry points' checks and the kernels.
#include "ktir_kv8_dev.h"

namespace ktir {

constexpr int64_t MASK_WORDS = 32;

// One wavefront for a token and query head: 64 keys at a time, one a lane, then the columns.
template <int CODE>
__global__ __launch_bounds__(64) void kv8_tree_row(const ktir_kv8_tree_attn_t T, int* err) {
  const ktir_kv8_attn_t& d = T.attn;
  const ktir_kv8_t& c = d.cache;
  __shared__ float qs[256], ps[64];
  __shared__ int64_t rows[64];
  __shared__ float vscale[64];
  const int l = threadIdx.x, D = (int)c.columns, shift = __builtin_ctz((uint32_t)c.page);
  const int64_t hq = blockIdx.y, head = hq / (d.q_heads / c.heads), tok = blockIdx.x;
  int64_t s, nth;
  const Seq q = seq_of_slot(d.batch, c.page, 1, 0, 0, tok, &s, &nth, err);
  if (nth < 0 || nth >= q.n_new) return;
  if (q.n_new > d.max_q || q.n_held > d.max_k) *err = OUT_OF_RANGE;
  if (nth >= d.max_q) return;
  const int64_t before = (int64_t)q.n_kv - q.n_new, keys = q.n_held < d.max_k ? q.n_held : d.max_k;
  int64_t lo = 0;
  if (d.window) {
    int64_t pos = ints(T.pos)[tok];
    pos = pos < before ? before : pos;
    lo = pos - d.window + 1 > 0 ? pos - d.window + 1 : 0;
  }
  int64_t least = d.window && before - d.window + 1 > 0 ? before - d.window + 1 : 0;
  for (int x = l; x < D; x += 64) qs[x] = load_elem(d.q.ptr, tok * d.q.tok + hq * d.q.head + x, d.dtype);
  __syncthreads();
  float m = -__builtin_inff(), sum = 0.f, acc[4] = {};
  for (int64_t base = least; base < keys; base += 64) {
    const int64_t j = base + l, bit = j - before;
    bool see = j < keys && (bit < 0 ? j >= lo : bit < 32 * T.words && (ints(T.mask)[tok * T.mask_row + bit / 32] >> (bit & 31) & 1));
    float sc = -__builtin_inff();
    rows[l] = 0;
    vscale[l] = 0.f;
    if (see) {
      int64_t page = ints(d.batch.table)[s * d.batch.table_row + (j >> shift)];
      if (page < 0 || page >= c.pages) *err = OUT_OF_RANGE, page = 0;
      const int64_t row = j & (c.page - 1);
      const KTIR_G(uint8_t)* kp = (const KTIR_G(uint8_t)*)c.k + page * c.k_page + row * c.k_tok + head * c.k_head;
      float t = 0.f;
      for (int x = 0; x < D; x += 4) {
        const uint32_t w = *(const KTIR_G(uint32_t)*)(kp + x);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          float v;
          if constexpr (CODE == KTIR_I8) v = (float)(int8_t)(w >> (8 * y));
          else v = y == 0 ? __builtin_amdgcn_cvt_f32_fp8(w, 0) : y == 1 ? __builtin_amdgcn_cvt_f32_fp8(w, 1) : y == 2 ? __builtin_amdgcn_cvt_f32_fp8(w, 2) : __builtin_amdgcn_cvt_f32_fp8(w, 3);
          t = __builtin_fmaf(qs[x + y], v, t);
        }
      }
      sc = t * ((const KTIR_G(float)*)c.k_scale)[page * c.ks_page + head * c.ks_head] * d.scale;
      rows[l] = page * c.v_page + row * c.v_tok + head * c.v_head;
      vscale[l] = ((const KTIR_G(float)*)c.v_scale)[page * c.vs_page + head * c.vs_head];
    }
    float top = sc;
    for (int o = 32; o; o >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o));
    const float now = __builtin_fmaxf(m, top);
    if (now == -__builtin_inff()) continue;
    const float p = see ? exp_f(sc - now) : 0.f, keep = exp_f(m - now);
    m = now;
    float t = p;
    for (int o = 32; o; o >>= 1) t += __shfl_xor(t, o);
    sum = sum * keep + t;
    ps[l] = p * vscale[l];
    __syncthreads();
    for (int i = 0; i < 4; ++i) acc[i] *= keep;
    const uint64_t some = __ballot(see);
    for (int r = 0; r < 64; ++r) {
      if (!(some >> r & 1)) continue;
      for (int i = 0; i < 4; ++i) {
        if (l + 64 * i >= D) break;
        const uint8_t w = ((const KTIR_G(uint8_t)*)c.v)[rows[r] + l + 64 * i];
        acc[i] += ps[r] * (CODE == KTIR_I8 ? (float)(int8_t)w : __builtin_amdgcn_cvt_f32_fp8(w, 0));
      }
    }
    __syncthreads();
  }
  const bool none = m == -__builtin_inff() && sum == 0.f;
  for (int i = 0; i < 4; ++i)
    if (l + 64 * i < D) store_elem(d.out.ptr, tok * d.out.tok + hq * d.out.head + l + 64 * i, d.dtype, none ? 0.f : acc[i] / sum);
  if (d.lse && l == 0) ((KTIR_G(float)*)d.lse)[tok * d.lse_tok + hq * d.lse_head] = none ? -__builtin_inff() : m + __logf(sum);
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
  d->attn.splits = 1;
  d->attn.ws_bytes = 0;
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
  if (!apart(out, mask) || !apart(out, pos) || (d->lse && (!apart(lse, mask) || !apart(lse, pos))))
    return set_error(KTIR_E_ARG, "%s: an output overlaps the mask or positions", ME);
  rc = ready(ME);
  if (rc != KTIR_OK) return rc;
  OnDevice on;
  if (!on.ok()) return set_error(KTIR_E_HIP, "%s: no device", ME);
  if (d->q_heads > 65535) return set_error(KTIR_E_UNSUPPORTED, "%s: %lld heads in one launch", ME, (long long)d->q_heads);
  const dim3 grid((unsigned)d->batch.tokens, (unsigned)d->q_heads);
  const hipStream_t st = stream_of(d->stream);
  if (d->cache.dtype == KTIR_I8) hipLaunchKernelGGL(kv8_tree_row<KTIR_I8>, grid, dim3(64), 0, st, *t, device_error_flag());
  else hipLaunchKernelGGL(kv8_tree_row<KTIR_E4M3>, grid, dim3(64), 0, st, *t, device_error_flag());
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}
