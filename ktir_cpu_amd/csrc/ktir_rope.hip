// Rotary positions: pairs of a head's columns rotated by an angle that grows
// with the token's position, y = (x0 c - x1 s, x1 c + x0 s).
//
// Bound: bytes, in and out once.  The angles of a token are made once for all its
// heads (remainder, sine and cosine in 64 bits), in LDS, and
// every vector of 16 bytes is loaded and stored once, two rows of loads ahead.
// Measured, f16 / bf16: 8192 tokens of 32 + 8 heads of 128, 168 MB, 31.9 us = 5.3 TB/s (31.7 with sine and cosine in 32 bits)
// (a copy of 256 MiB makes 5.4 here); 40 + 40 heads with 64 interleaved columns of
// 128, 168 MB, 36.2 us, 55.8 (of 39.4) with the columns behind rot as units of their own size;
// one thread per pair over all heads took 97 and 212 us.  One token: a launch, 4.1 us.
#include "ktir_rope_dev.h"

namespace ktir {

constexpr int ROPE_PAIRS = 2048;     // angles of a workgroup's tokens in LDS
constexpr int ROPE_TOKENS = 8;

// A workgroup has `per` tokens and, with several in y, a part of the heads.  Its
// threads first make the angles of the tokens together, then each takes one unit of
// columns over rows (token, head), R rows' loads ahead of the first's stores.
template <int DT, bool INTER, int V, int R, bool PAST>
__global__ __launch_bounds__(256) void rope_turn(const ktir_rope_t d, int per) {
  __shared__ __attribute__((aligned(16))) float cs[ROPE_PAIRS], sn[ROPE_PAIRS];
  __shared__ int live[ROPE_TOKENS];
  const int half = (int)(d.rot / 2), rot = (int)d.rot, columns = (int)d.columns, pairs = half / V;
  const bool tail = d.in.ptr != d.out.ptr || (d.heads2 && d.in2.ptr != d.out2.ptr);
  const int units = pairs + (tail ? (columns - rot + 2 * V - 1) / (2 * V) : 0);
  const int64_t t0 = (int64_t)blockIdx.x * per;
  const int tokens = (int)(d.tokens - t0 < per ? d.tokens - t0 : per), heads = (int)(d.heads + d.heads2);
  const int wide = units < 256 ? units : 256, step = 256 / wide;      // columns side by side, rows side by side
  const int tid = threadIdx.x, u0 = tid % wide, stride = step * (int)gridDim.y, total = tokens * heads;

  for (int i = tid; i < tokens * half; i += 256) {
    const int t = i / half;
    const int64_t pos = rope_pos(d, t0 + t);
    rope_angle(d, pos < 0 ? 0 : pos, i - t * half, &cs[i], &sn[i]);
  }
  for (int t = tid; t < tokens; t += 256) live[t] = rope_pos(d, t0 + t) >= 0;
  __syncthreads();
  if (tid >= wide * step) return;
  for (int u = u0; u < units; u += wide) {
    int a, b;
    rope_columns<INTER, V>(u, pairs, half, rot, &a, &b);
    const bool two = b < columns;            // the last unit behind rot may be half one
    if (!two) b = a;
    int row = (int)blockIdx.y * step + tid / wide, t = 0, h = row;
    while (row < total) {
      RopeRaw<DT, V> r[R];
      int at[R];
      int64_t to[R];
      uint64_t ptr[R];
#pragma unroll
      for (int k = 0; k < R; ++k) {
        while (h >= heads) {
          h -= heads;
          ++t;
        }
        const bool second = h >= d.heads, on = row < total && live[t < tokens ? t : 0];
        const ktir_rows3_t &in = second ? d.in2 : d.in, &out = second ? d.out2 : d.out;
        const int64_t hh = second ? h - d.heads : h;
        to[k] = (t0 + t) * out.tok + hh * out.head;
        ptr[k] = on && (u < pairs || in.ptr != out.ptr) ? out.ptr : 0;
        at[k] = t * half + u * V;
        if (ptr[k]) {
          const int64_t e = (t0 + t) * in.tok + hh * in.head;
          rope_load<DT, V, PAST>(in.ptr, e + a, e + b, r[k]);
        }
        row += stride;
        h += stride;
      }
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (!ptr[k]) continue;
        if (u < pairs) {
          __attribute__((aligned(16))) float c[V], s[V];
          if constexpr (V > 1) {                             // half and so every unit's angles: multiples of 4
#pragma unroll
            for (int i = 0; i < V; i += 4) {
              *(f4_t*)(c + i) = *(const f4_t*)&cs[at[k] + i];
              *(f4_t*)(s + i) = *(const f4_t*)&sn[at[k] + i];
            }
          } else {
            c[0] = cs[at[k]];
            s[0] = sn[at[k]];
          }
          rope_turn_raw<DT, INTER, V>(r[k], c, s);
        }
        rope_store<DT, V>(ptr[k], to[k] + a, to[k] + b, r[k], two);
      }
    }
  }
}

// whether every vector of V values of a tensor starts on a 16-byte bound
static bool wide_rows(const ktir_rows3_t& r, int64_t tokens, int64_t heads, int V) {
  return !(r.ptr & 15) && (tokens == 1 || r.tok % V == 0) && (heads == 1 || r.head % V == 0);
}

template <int DT, int V>
static void rope_go(const ktir_rope_t& d, hipStream_t st) {
  const int64_t half = d.rot / 2, units = half / V + (d.columns - d.rot + 2 * V - 1) / (2 * V), heads = d.heads + d.heads2;
  int64_t per = d.tokens / 1024;
  per = per > ROPE_TOKENS ? ROPE_TOKENS : per < 1 ? 1 : per;
  if (per * half > ROPE_PAIRS) per = ROPE_PAIRS / half;
  const int64_t blocks = (d.tokens + per - 1) / per, step = 256 / (units < 256 ? units : 256);
  constexpr int R = 2;
  // few tokens: one row of units a thread
  int64_t y = 1;
  if (blocks < 512) {
    y = (per * heads + step - 1) / step;
    const int64_t most = (1024 + blocks - 1) / blocks;
    y = y > most ? most : y;
  }
  const dim3 grid((unsigned)blocks, (unsigned)y);
  // Inputs and outputs past 64 MB, twice what the L2s hold: the inputs, which are done with, are read
  // past the caches and leave them to the outputs.  Turned, appended and attended to by 32 / 8 heads of 128:
  // 8192 tokens (168 MB) 53.2 -> 49.5 us and 611 -> 610 with attention, 5120 35.3 -> 31.3 and 290.8 -> 289.0,
  // 3584 (73 MB) 24.1 -> 23.8 and 149.9 -> 148.5, but 2048 (42 MB) 16.1 -> 17.9 and 83.1 -> 84.9.  Outputs stored
  // past the caches make the turn as fast, but attention then reads them from HBM: 615.7 with 8192 tokens.
  // In place the lines are written again at once: 4096 tokens 15.8 as they are, 19.0 past the caches.
  constexpr bool WIDE = V > 1;
  const bool past = WIDE && d.in.ptr != d.out.ptr && (!d.heads2 || d.in2.ptr != d.out2.ptr) && 2 * d.tokens * heads * d.columns * (DT == KTIR_F32 ? 4 : 2) > (int64_t)64 << 20;
  if (d.interleaved) {
    if (past) hipLaunchKernelGGL((rope_turn<DT, true, V, R, WIDE>), grid, dim3(256), 0, st, d, (int)per);
    else hipLaunchKernelGGL((rope_turn<DT, true, V, R, false>), grid, dim3(256), 0, st, d, (int)per);
  } else {
    if (past) hipLaunchKernelGGL((rope_turn<DT, false, V, R, WIDE>), grid, dim3(256), 0, st, d, (int)per);
    else hipLaunchKernelGGL((rope_turn<DT, false, V, R, false>), grid, dim3(256), 0, st, d, (int)per);
  }
}

static int check_tensors(const ktir_rope_t& d) {
  constexpr const char* ME = "ktir_launch_rope";
  int rc = check_rows3(ME, d.in, d.tokens, d.heads, d.columns, false);
  if (rc == KTIR_OK) rc = check_rows3(ME, d.out, d.tokens, d.heads, d.columns, true);
  if (rc == KTIR_OK && d.heads2) rc = check_rows3(ME, d.in2, d.tokens, d.heads2, d.columns, false);
  if (rc == KTIR_OK && d.heads2) rc = check_rows3(ME, d.out2, d.tokens, d.heads2, d.columns, true);
  if (rc != KTIR_OK) return rc;
  auto rows = [&](const ktir_rows3_t& r, int64_t heads) { return rows_of(r, d.tokens, heads, d.columns, d.dtype == KTIR_F32 ? 4 : 2); };
  const Strided in = rows(d.in, d.heads), out = rows(d.out, d.heads), in2 = rows(d.in2, d.heads2), out2 = rows(d.out2, d.heads2);
  bool good = same(in, out) || apart(in, out);
  if (d.heads2) good = good && (same(in2, out2) || apart(in2, out2)) && apart(out, in2) && apart(out2, in) && apart(out, out2);
  if (!good) return set_error(KTIR_E_ARG, "%s: an output overlaps a tensor that it is not", ME);
  const Strided pos(d.pos, d.tokens * (d.pos_dtype == KTIR_I64 ? 8 : 4)), freq(d.freq, d.rot / 2 * 8);
  good = apart(out, pos) && apart(out, freq) && (!d.heads2 || (apart(out2, pos) && apart(out2, freq)));
  return good ? KTIR_OK : set_error(KTIR_E_ARG, "%s: an output overlaps the positions or frequencies", ME);
}

}  // namespace ktir

using namespace ktir;

extern "C" int ktir_launch_rope(const ktir_rope_t* d) {
  if (!d) return set_error(KTIR_E_ARG, "ktir_launch_rope: no descriptor");
  if (d->tokens < 0 || d->tokens > INT32_MAX || d->heads < 1 || d->heads2 < 0 || d->columns < 1 || d->columns > 4096 || d->heads > 65536 || d->heads2 > 65536)
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
  int rc = check_tensors(*d);
  if (rc == KTIR_OK) rc = ready("ktir_launch_rope");
  if (rc != KTIR_OK) return rc;
  OnDevice on;
  if (!on.ok()) return set_error(KTIR_E_HIP, "ktir_launch_rope: no device");
  const int V = d->dtype == KTIR_F32 ? 4 : 8;
  bool wide = (d->rot / 2) % V == 0 && (d->columns - d->rot) % V == 0 && wide_rows(d->in, d->tokens, d->heads, V) &&
              wide_rows(d->out, d->tokens, d->heads, V);
  if (d->heads2) wide = wide && wide_rows(d->in2, d->tokens, d->heads2, V) && wide_rows(d->out2, d->tokens, d->heads2, V);
  const hipStream_t st = stream_of(d->stream);
  switch (d->dtype) {
    case KTIR_F32: wide ? rope_go<KTIR_F32, 4>(*d, st) : rope_go<KTIR_F32, 1>(*d, st); break;
    case KTIR_F16: wide ? rope_go<KTIR_F16, 8>(*d, st) : rope_go<KTIR_F16, 1>(*d, st); break;
    default: wide ? rope_go<KTIR_BF16, 8>(*d, st) : rope_go<KTIR_BF16, 1>(*d, st);
  }
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}
