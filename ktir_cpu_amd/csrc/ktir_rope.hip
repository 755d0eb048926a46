// Rotary positions: pairs of a head's columns rotated by an angle that grows
// with the token's position, y = (x0 c - x1 s, x1 c + x0 s).
#include <climits>
#include "ktir_serve.h"

namespace ktir {

// cosine and sine of token t's pair i, times the amplitude.  The angle passes
// 2^20 radians at far positions, where f32 holds it to a sixteenth: the product
// and its remainder of whole turns are f64, what is left is f32 (2^-25 turns).
__device__ __forceinline__ void rope_angle(const ktir_rope_t& d, int64_t pos, int i, float* c, float* s) {
  double turns = (double)pos * ((const KTIR_G(double)*)d.freq)[i] * 0.15915494309189533577;
  turns -= rint(turns);
  float sn, cs;
  sincospif((float)(2.0 * turns), &sn, &cs);
  const float amp = (float)d.amplitude;
  *c = cs * amp;
  *s = d.inverse ? -(sn * amp) : sn * amp;
}

__device__ __forceinline__ int64_t rope_pos(const ktir_rope_t& d, int64_t t) {
  return d.pos_dtype == KTIR_I64 ? ((const KTIR_G(int64_t)*)d.pos)[t] : (int64_t)ints(d.pos)[t];
}

__global__ __launch_bounds__(256) void rope_plain(const ktir_rope_t d) {
  const int64_t half = d.rot / 2, per = half + (d.columns - d.rot), total = d.tokens * per;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (int64_t)gridDim.x * 256) {
    const int64_t t = at / per, i = at - t * per, pos = rope_pos(d, t);
    if (pos < 0) continue;
    float c = 1.f, s = 0.f;
    if (i < half) rope_angle(d, pos, (int)i, &c, &s);
    for (int64_t h = 0; h < d.heads + d.heads2; ++h) {
      const ktir_rows3_t &in = h < d.heads ? d.in : d.in2, &out = h < d.heads ? d.out : d.out2;
      const int64_t hh = h < d.heads ? h : h - d.heads, e = t * in.tok + hh * in.head, o = t * out.tok + hh * out.head;
      if (i >= half) {
        const int64_t x = d.rot + (i - half);
        if (in.ptr != out.ptr) store_elem(out.ptr, o + x, d.dtype, load_elem(in.ptr, e + x, d.dtype));
        continue;
      }
      const int64_t x0 = d.interleaved ? 2 * i : i, x1 = d.interleaved ? 2 * i + 1 : i + half;
      const float a = load_elem(in.ptr, e + x0, d.dtype), b = load_elem(in.ptr, e + x1, d.dtype);
      store_elem(out.ptr, o + x0, d.dtype, __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)));
      store_elem(out.ptr, o + x1, d.dtype, __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s)));
    }
  }
}

static int check_pair(const ktir_rope_t& d, const ktir_rows3_t& in, const ktir_rows3_t& out, int64_t heads) {
  int rc = check_rows3("ktir_launch_rope", in, d.tokens, heads, d.columns, false);
  if (rc == KTIR_OK) rc = check_rows3("ktir_launch_rope", out, d.tokens, heads, d.columns, true);
  if (rc != KTIR_OK) return rc;
  if (in.ptr == out.ptr && (in.tok == out.tok || d.tokens == 1) && (in.head == out.head || heads == 1)) return KTIR_OK;
  const int e = d.dtype == KTIR_F32 ? 4 : 2;
  if (in.ptr < end_of(out, d.tokens, heads, d.columns, e) && out.ptr < end_of(in, d.tokens, heads, d.columns, e))
    return set_error(KTIR_E_ARG, "ktir_launch_rope: an output overlaps its input without being it");
  return KTIR_OK;
}

}  // namespace ktir

using namespace ktir;

extern "C" int ktir_launch_rope(const ktir_rope_t* d) {
  if (!d) return set_error(KTIR_E_ARG, "ktir_launch_rope: no descriptor");
  if (d->tokens < 0 || d->heads < 1 || d->heads2 < 0 || d->columns < 1 || d->columns > 4096 || d->heads > 65536 || d->heads2 > 65536)
    return set_error(KTIR_E_ARG, "ktir_launch_rope: %lld tokens, %lld and %lld heads of %lld columns", (long long)d->tokens,
                     (long long)d->heads, (long long)d->heads2, (long long)d->columns);
  if (d->rot < 2 || d->rot > d->columns || (d->rot & 1))
    return set_error(KTIR_E_ARG, "ktir_launch_rope: %lld of %lld columns rotated (an even number of them)", (long long)d->rot,
                     (long long)d->columns);
  if (d->dtype != KTIR_F16 && d->dtype != KTIR_BF16 && d->dtype != KTIR_F32)
    return set_error(KTIR_E_UNSUPPORTED, "ktir_launch_rope: dtype %d", d->dtype);
  if (d->pos_dtype != KTIR_I32 && d->pos_dtype != KTIR_I64)
    return set_error(KTIR_E_UNSUPPORTED, "ktir_launch_rope: positions of dtype %d", d->pos_dtype);
  if (!(d->amplitude - d->amplitude == 0.0)) return set_error(KTIR_E_ARG, "ktir_launch_rope: amplitude is not finite");
  if (d->tokens == 0) return KTIR_OK;
  if (!d->pos || !d->freq || (d->freq & 7)) return set_error(KTIR_E_ARG, "ktir_launch_rope: positions or frequencies missing");
  int rc = check_pair(*d, d->in, d->out, d->heads);
  if (rc == KTIR_OK && d->heads2) rc = check_pair(*d, d->in2, d->out2, d->heads2);
  if (rc == KTIR_OK) rc = ready("ktir_launch_rope");
  if (rc != KTIR_OK) return rc;
  OnDevice on;
  if (!on.ok()) return set_error(KTIR_E_HIP, "ktir_launch_rope: no device");
  const int64_t total = d->tokens * (d->rot / 2 + d->columns - d->rot), blocks = (total + 255) / 256;
  hipLaunchKernelGGL(rope_plain, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, stream_of(d->stream), *d);
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}
