// Attention over the key / value cache in 8 bits.
#include "ktir_attn_common.h"
#include "ktir_serve.h"

namespace ktir {

template <int CODE>
__device__ __forceinline__ float kv8_value(uint8_t c) {
  if constexpr (CODE == KTIR_I8) return (float)(int8_t)c;
  else return __builtin_amdgcn_cvt_f32_fp8(c, 0);
}

// One wavefront per token and query head, one key per lane, online softmax over
// blocks of 64 keys; everything in f32.
template <int CODE>
__global__ __launch_bounds__(64) void kv8_attn_plain(const ktir_kv8_attn_t d, int* err) {
  __shared__ float q[256], p[64];
  __shared__ uint64_t vrow[64];
  const ktir_kv8_t& c = d.cache;
  const int l = threadIdx.x, D = (int)c.columns;
  const int64_t t = blockIdx.x, head = blockIdx.y;
  int64_t s = -1;
  for (int64_t base = 0; base < d.batch.seqs && s < 0; base += 64) {
    const bool mine = base + l < d.batch.seqs && ints(d.batch.q_start)[base + l] <= t && ints(d.batch.q_start)[base + l + 1] > t;
    const uint64_t found = __ballot(mine);
    if (found) s = base + __builtin_ctzll(found);
  }
  if (s < 0) return;
  const Seq q_ = seq_of(d.batch, c.page, s, err);
  const int64_t i = t - q_.start, pos = (int64_t)q_.n_kv - q_.n_new + i;
  if (i < 0 || i >= q_.n_new) return;
  int64_t keys = q_.n_held;
  if (i >= d.max_q || keys > d.max_k) {
    *err = OUT_OF_RANGE;
    if (i >= d.max_q) return;
    keys = d.max_k;
  }
  const int64_t hi = d.causal && pos + 1 < keys ? pos + 1 : keys;
  int64_t lo = d.window && pos - d.window + 1 > 0 ? pos - d.window + 1 : 0;
  const int64_t kv = head / (d.q_heads / c.heads);
  for (int x = l; x < D; x += 64) q[x] = load_elem(d.q.ptr, t * d.q.tok + head * d.q.head + x, d.dtype);
  __syncthreads();
  float m = -__builtin_inff(), sum = 0.f, acc[4] = {};
  for (; lo < hi; lo += 64) {
    const int64_t j = lo + l;
    float w = -__builtin_inff(), vs = 0.f;
    vrow[l] = 0;
    if (j < hi) {
      int64_t at = ints(d.batch.table)[s * d.batch.table_row + j / c.page];
      if (at < 0 || at >= c.pages) {
        *err = OUT_OF_RANGE;
        at = 0;
      }
      const int64_t r = j % c.page;
      const KTIR_G(uint8_t)* k = (const KTIR_G(uint8_t)*)c.k + at * c.k_page + r * c.k_tok + kv * c.k_head;
      float dot = 0.f;
      for (int x = 0; x < D; ++x) dot = __builtin_fmaf(q[x], kv8_value<CODE>(k[x]), dot);
      w = dot * (d.scale * ((const KTIR_G(float)*)c.k_scale)[at * c.ks_page + kv * c.ks_head]);
      vs = ((const KTIR_G(float)*)c.v_scale)[at * c.vs_page + kv * c.vs_head];
      vrow[l] = c.v + at * c.v_page + r * c.v_tok + kv * c.v_head;
    }
    float top = w;
    for (int o = 32; o; o >>= 1) top = fmax_nan(top, __shfl_xor(top, o));
    const float m2 = fmax_nan(m, top), alpha = m == m2 ? 1.f : __expf(m - m2), e = j < hi ? __expf(w - m2) : 0.f;
    float part = e;
    for (int o = 32; o; o >>= 1) part += __shfl_xor(part, o);
    sum = sum * alpha + part;
    m = m2;
    p[l] = j < hi ? e * vs : 0.f;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int x = l + 64 * k;
      acc[k] *= alpha;
      if (x < D)
        for (int n = 0; n < 64 && lo + n < hi; ++n) acc[k] = __builtin_fmaf(p[n], kv8_value<CODE>(((const KTIR_G(uint8_t)*)vrow[n])[x]), acc[k]);
    }
    __syncthreads();
  }
  const bool none = (d.window && pos - d.window + 1 > 0 ? pos - d.window + 1 : 0) >= hi;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (l + 64 * k < D) store_elem(d.out.ptr, t * d.out.tok + head * d.out.head + l + 64 * k, d.dtype, none ? 0.f : acc[k] / sum);
  if (d.lse && l == 0) ((KTIR_G(float)*)d.lse)[t * d.lse_tok + head * d.lse_head] = none ? -__builtin_inff() : m + logf(sum);
}

static int check_attn(const char* what, const ktir_kv8_attn_t& d) {
  if (d.dtype != KTIR_F16 && d.dtype != KTIR_BF16) return set_error(KTIR_E_UNSUPPORTED, "%s: dtype %d", what, d.dtype);
  int rc = check_kv8(what, d.cache, false);
  if (rc == KTIR_OK) rc = check_batch(what, d.batch, d.cache);
  if (rc != KTIR_OK) return rc;
  if (d.q_heads < 1 || d.q_heads % d.cache.heads || d.q_heads > 65536)
    return set_error(KTIR_E_ARG, "%s: %lld query heads over %lld", what, (long long)d.q_heads, (long long)d.cache.heads);
  if (d.max_q < 0 || d.max_k < 0 || d.max_k > INT32_MAX - 65536) return set_error(KTIR_E_ARG, "%s: bounds %lld and %lld", what, (long long)d.max_q, (long long)d.max_k);
  if (d.window < 0 || (d.window && !d.causal)) return set_error(KTIR_E_ARG, "%s: window %lld", what, (long long)d.window);
  if (!(d.scale - d.scale == 0.f)) return set_error(KTIR_E_ARG, "%s: scale is not finite", what);
  if (d.splits < 0) return set_error(KTIR_E_ARG, "%s: %d splits", what, d.splits);
  return KTIR_OK;
}

}  // namespace ktir

using namespace ktir;

extern "C" int ktir_kv8_attention_plan(ktir_kv8_attn_t* d) {
  constexpr const char* ME = "ktir_kv8_attention_plan";
  if (!d) return set_error(KTIR_E_ARG, "%s: no descriptor", ME);
  const int rc = check_attn(ME, *d);
  if (rc != KTIR_OK) return rc;
  d->splits = 1;
  d->ws_bytes = 0;
  return KTIR_OK;
}

extern "C" int ktir_launch_kv8_attention(const ktir_kv8_attn_t* d) {
  constexpr const char* ME = "ktir_launch_kv8_attention";
  if (!d) return set_error(KTIR_E_ARG, "%s: no descriptor", ME);
  int rc = check_attn(ME, *d);
  if (rc != KTIR_OK || d->batch.seqs == 0 || d->batch.tokens == 0) return rc;
  rc = check_rows3(ME, d->q, d->batch.tokens, d->q_heads, d->cache.columns, false);
  if (rc == KTIR_OK) rc = check_rows3(ME, d->out, d->batch.tokens, d->q_heads, d->cache.columns, true);
  if (rc == KTIR_OK && d->lse) {
    const ktir_rows3_t lse = {d->lse, d->lse_tok, d->lse_head};
    rc = d->lse & 3 ? set_error(KTIR_E_ARG, "%s: lse off 4-byte bounds", ME) : check_rows3(ME, lse, d->batch.tokens, d->q_heads, 1, true);
  }
  if (rc == KTIR_OK) rc = ready(ME);
  if (rc != KTIR_OK) return rc;
  OnDevice on;
  if (!on.ok()) return set_error(KTIR_E_HIP, "%s: no device", ME);
  const dim3 grid((unsigned)d->batch.tokens, (unsigned)d->q_heads);
  if (d->cache.dtype == KTIR_I8) hipLaunchKernelGGL(kv8_attn_plain<KTIR_I8>, grid, dim3(64), 0, stream_of(d->stream), *d, device_error_flag());
  else hipLaunchKernelGGL(kv8_attn_plain<KTIR_E4M3>, grid, dim3(64), 0, stream_of(d->stream), *d, device_error_flag());
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}
