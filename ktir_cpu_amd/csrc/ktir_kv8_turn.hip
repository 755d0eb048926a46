// Rotary positions and append to the 8-bit cache in one launch.
#include "ktir_kv8_codes.h"
#include "ktir_rope_dev.h"

namespace ktir {

template <int DT>
__device__ __forceinline__ float turn_get(uint64_t ptr, int64_t e) {
  return load_elem(ptr, e, DT);
}

// A workgroup for each page that new tokens fall in, and head of the queries, keys or values (y).
template <int CODE, int DT>
__global__ __launch_bounds__(256) void kv8_turn(const ktir_kv8_rope_append_t d, int* err) {
  __shared__ float tops[4];
  __shared__ int odd[4];
  const ktir_kv8_t& c = d.cache;
  const int tid = threadIdx.x, y = blockIdx.y, D = (int)c.columns, half = (int)d.rot / 2, rot = (int)d.rot;
  const int kind = y < d.q_heads ? 0 : y < d.q_heads + c.heads ? 1 : 2;          // queries, keys, values
  const int64_t head = y - (kind ? d.q_heads : 0) - (kind == 2 ? c.heads : 0);
  const int shift = __builtin_ctz((uint32_t)c.page);
  int64_t s, nth;
  const Seq q = seq_of_slot(d.batch, c.page, 1, shift, 2, blockIdx.x, &s, &nth, err);
  if (nth < 0) return;
  const int64_t pos0 = (int64_t)q.n_kv - q.n_new, from = pos0 < 0 ? 0 : pos0;
  const int64_t p = (from >> shift) + nth;
  const int64_t lo = p << shift < from ? from : p << shift, hi = (p + 1) << shift < q.n_held ? (p + 1) << shift : q.n_held;
  if (lo >= hi) return;
  const int64_t at = ints(d.batch.table)[s * d.batch.table_row + p];
  if (at < 0 || at >= c.pages) {
    *err = OUT_OF_RANGE;
    return;
  }
  const int n = (int)(hi - lo), r0 = (int)(lo & (c.page - 1));
  const int64_t t0 = q.start + lo - pos0;
  const ktir_rows3_t& in = kind == 0 ? d.q : kind == 1 ? d.k : d.v;

  auto angle = [&](int r, int i, float* cs, float* sn) {
    int64_t pos = d.pos ? rope_pos(d.pos, d.pos_dtype, t0 + r) : lo + r;
    if (pos < 0) {
      *err = OUT_OF_RANGE;
      pos = 0;
    }
    rope_angle(d.freq, d.amplitude, false, pos, i, cs, sn);
  };
  auto first_of = [&](int i) { return d.interleaved ? 2 * i : i; };
  const int gap = d.interleaved ? 1 : half;
  // the pair i of row r, turned
  auto pair = [&](int r, int i, float* u, float* v) {
    const int64_t e = (t0 + r) * in.tok + head * in.head + first_of(i);
    const float a = turn_get<DT>(in.ptr, e), b = turn_get<DT>(in.ptr, e + gap);
    float cs, sn;
    angle(r, i, &cs, &sn);
    *u = __fsub_rn(__fmul_rn(a, cs), __fmul_rn(b, sn));
    *v = __fadd_rn(__fmul_rn(b, cs), __fmul_rn(a, sn));
  };
  const int units = half + D - rot;                // pairs, then columns behind rot
  if (kind == 0) {
    for (int x = tid; x < n * units; x += 256) {
      const int r = x / units, i = x - r * units;
      const int64_t o = (t0 + r) * d.q_out.tok + head * d.q_out.head;
      if (i < half) {
        float u, v;
        pair(r, i, &u, &v);
        store_elem(d.q_out.ptr, o + first_of(i), DT, u);
        store_elem(d.q_out.ptr, o + first_of(i) + gap, DT, v);
      } else {
        const int col = rot + i - half;
        store_elem(d.q_out.ptr, o + col, DT, turn_get<DT>(in.ptr, (t0 + r) * in.tok + head * in.head + col));
      }
    }
    return;
  }
  // column x of row r
  auto value = [&](int r, int x) {
    if (kind == 2 || x >= rot) return turn_get<DT>(in.ptr, (t0 + r) * in.tok + head * in.head + x);
    const int i = d.interleaved ? x / 2 : x < half ? x : x - half;
    float u, v;
    pair(r, i, &u, &v);
    return x == first_of(i) ? u : v;
  };
  float top = 0.f;
  bool finite = true;
  for (int x = tid; x < n * D; x += 256) {
    const float v = __builtin_fabsf(value(x / D, x % D));
    top = __builtin_fmaxf(top, v);
    finite = finite && v < __builtin_inff();
  }
  for (int o = 32; o; o >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o));
  finite = __all(finite);
  if ((tid & 63) == 0) tops[tid >> 6] = top, odd[tid >> 6] = !finite;
  const bool is_v = kind == 2;
  KTIR_G(uint8_t)* codes = (KTIR_G(uint8_t)*)(is_v ? c.v + at * c.v_page + head * c.v_head : c.k + at * c.k_page + head * c.k_head);
  const int64_t tok = is_v ? c.v_tok : c.k_tok;
  KTIR_G(float)* scale = is_v ? (KTIR_G(float)*)c.v_scale + at * c.vs_page + head * c.vs_head
                              : (KTIR_G(float)*)c.k_scale + at * c.ks_page + head * c.ks_head;
  const float before = r0 ? *scale : 0.f;
  __syncthreads();
  for (int i = 0; i < 4; ++i) {
    top = __builtin_fmaxf(top, tops[i]);
    finite = finite && !odd[i];
  }
  float now = __builtin_fmaxf(top * PER_TOP<CODE>, LEAST_SCALE);
  if (!(now >= before)) now = before;                     // a page that was NaN stays so
  if (!finite) now = __builtin_nanf("");
  const bool nan = !(now < __builtin_inff());
  const float inv = 1.f / now;
  auto put = [&](int row, int x, float v) {
    float y[4] = {v, 0.f, 0.f, 0.f};
    codes[row * tok + x] = (uint8_t)codes4<CODE, CODE == KTIR_E4M3>(y);
  };
  if (now > before)
    for (int x = tid; x < r0 * D; x += 256) {
      float y[4];
      values4<CODE>(codes[x / D * tok + x % D], y);
      put(x / D, x % D, y[0] * (before * inv));
    }
  for (int x = tid; x < n * D; x += 256) put(r0 + x / D, x % D, nan ? 0.f : value(x / D, x % D) * inv);
  if (tid == 0) *scale = now;
}

}  // namespace ktir

using namespace ktir;

extern "C" int ktir_launch_kv8_rope_append(const ktir_kv8_rope_append_t* d) {
  constexpr const char* ME = "ktir_launch_kv8_rope_append";
  if (!d) return set_error(KTIR_E_ARG, "%s: no descriptor", ME);
  if (d->dtype != KTIR_F16 && d->dtype != KTIR_BF16) return set_error(KTIR_E_UNSUPPORTED, "%s: dtype %d", ME, d->dtype);
  int rc = check_kv8(ME, d->cache, true);
  if (rc == KTIR_OK) rc = check_batch(ME, d->batch, d->cache);
  if (rc != KTIR_OK) return rc;
  const int64_t tokens = d->batch.tokens, columns = d->cache.columns;
  if (d->q_heads < 1 || d->q_heads > 65536) return set_error(KTIR_E_ARG, "%s: %lld query heads", ME, (long long)d->q_heads);
  if (d->rot < 2 || d->rot > columns || (d->rot & 1))
    return set_error(KTIR_E_ARG, "%s: %lld of %lld columns rotated (an even number of them)", ME, (long long)d->rot, (long long)columns);
  if (d->pos && d->pos_dtype != KTIR_I32 && d->pos_dtype != KTIR_I64)
    return set_error(KTIR_E_UNSUPPORTED, "%s: positions of dtype %d", ME, d->pos_dtype);
  if (!(d->amplitude - d->amplitude == 0.0)) return set_error(KTIR_E_ARG, "%s: amplitude is not finite", ME);
  if (d->batch.seqs == 0 || tokens == 0) return KTIR_OK;
  const int pos_bytes = d->pos_dtype == KTIR_I64 ? 8 : 4;
  if (!d->freq || (d->freq & 7) || (d->pos & (pos_bytes - 1))) return set_error(KTIR_E_ARG, "%s: positions or frequencies missing or off their bounds", ME);
  rc = check_rows3(ME, d->q, tokens, d->q_heads, columns, false);
  if (rc == KTIR_OK) rc = check_rows3(ME, d->q_out, tokens, d->q_heads, columns, true);
  if (rc == KTIR_OK) rc = check_rows3(ME, d->k, tokens, d->cache.heads, columns, false);
  if (rc == KTIR_OK) rc = check_rows3(ME, d->v, tokens, d->cache.heads, columns, false);
  if (rc != KTIR_OK) return rc;
  const BatchParts batch(d->batch);
  const CacheParts cache(d->cache);
  const Strided q = rows_of(d->q, tokens, d->q_heads, columns, 2), q_out = rows_of(d->q_out, tokens, d->q_heads, columns, 2);
  const Strided k = rows_of(d->k, tokens, d->cache.heads, columns, 2), v = rows_of(d->v, tokens, d->cache.heads, columns, 2);
  const Strided freq(d->freq, d->rot / 2 * 8), pos = d->pos ? Strided(d->pos, tokens * pos_bytes) : freq;
  if (!(same(q, q_out) || apart(q, q_out)) || !apart(q_out, k) || !apart(q_out, v) || !apart(q_out, freq) || !apart(q_out, pos) || !batch.clear_of(q_out))
    return set_error(KTIR_E_ARG, "%s: an output overlaps a tensor that it is not", ME);
  for (const Strided& out : cache.x) {
    if (!apart(out, q) || !apart(out, q_out) || !apart(out, k) || !apart(out, v)) return set_error(KTIR_E_ARG, "%s: the cache overlaps the queries, keys or values", ME);
    if (!batch.clear_of(out) || !apart(out, freq) || !apart(out, pos)) return set_error(KTIR_E_ARG, "%s: the cache overlaps the table, offsets, lengths, positions or frequencies", ME);
  }
  rc = ready(ME);
  if (rc != KTIR_OK) return rc;
  OnDevice on;
  if (!on.ok()) return set_error(KTIR_E_HIP, "%s: no device", ME);
  // a sequence's n new tokens touch at most floor(n / page) + 2 pages
  const int64_t slots = tokens / d->cache.page + 2 * d->batch.seqs, all = d->q_heads + 2 * d->cache.heads;
  if (slots > INT32_MAX || all > 65535) return set_error(KTIR_E_UNSUPPORTED, "%s: %lld pages, %lld heads in one launch", ME, (long long)slots, (long long)all);
  const hipStream_t st = stream_of(d->stream);
  const dim3 grid((unsigned)slots, (unsigned)all);
  if (d->cache.dtype == KTIR_I8) {
    if (d->dtype == KTIR_BF16) hipLaunchKernelGGL((kv8_turn<KTIR_I8, KTIR_BF16>), grid, dim3(256), 0, st, *d, device_error_flag());
    else hipLaunchKernelGGL((kv8_turn<KTIR_I8, KTIR_F16>), grid, dim3(256), 0, st, *d, device_error_flag());
  } else {
    if (d->dtype == KTIR_BF16) hipLaunchKernelGGL((kv8_turn<KTIR_E4M3, KTIR_BF16>), grid, dim3(256), 0, st, *d, device_error_flag());
    else hipLaunchKernelGGL((kv8_turn<KTIR_E4M3, KTIR_F16>), grid, dim3(256), 0, st, *d, device_error_flag());
  }
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}
