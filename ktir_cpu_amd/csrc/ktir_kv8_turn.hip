// Rotary positions and append to the 8-bit cache in one launch.
//
// Two kinds of workgroups.  One turns queries: a few tokens, whose angles it makes once (in 64
// bits) for all heads, two rows of 16-byte loads a thread ahead of the stores.  The other has a page that new
// tokens fall in, and K or V: a wavefront a head (four where a page's part of a head is more
// than 256 units of 16 columns), its turned values in f32 registers from the maximum to the
// codes.  A unit of K loads its 16 columns and those that they are turned with, which a neighbour
// has just loaded: all layouts of pairs then store 16 codes at once.
#include "ktir_kv8_codes.h"
#include "ktir_rope_dev.h"

namespace ktir {

constexpr int TURN_PAIRS = 2048;     // angles in LDS
constexpr int TURN_TOKENS = 8;       // of a workgroup that turns queries
constexpr int TURN_KEPT = 4;         // units of 16 columns that a thread keeps

struct Angles {
  uint64_t freq;
  double amplitude;
  bool inverse;
};

// how a launch is cut: workgroups of keys and values first, then those of queries
struct TurnGrid {
  int kv;              // workgroups for a page: of keys, then as many of values
  int slots;           // pages
  int per, parts;      // tokens of a workgroup of queries, workgroups that share their heads
};

// ---- queries -----------------------------------------------------------------

template <int DT, bool INTER, int V, bool PAST>
__device__ __forceinline__ void turn_queries(const ktir_kv8_rope_append_t& d, int block, const TurnGrid& g, float* cs, float* sn, int64_t* place, int* err) {
  constexpr int R = 2;
  const int tid = threadIdx.x, half = (int)d.rot / 2, rot = (int)d.rot, columns = (int)d.cache.columns, pairs = half / V;
  const int64_t t0 = (int64_t)(block / g.parts) * g.per;
  const int tokens = (int)(d.batch.tokens - t0 < g.per ? d.batch.tokens - t0 : g.per), heads = (int)d.q_heads;
  // a token's position, or -1 where it is not stored
  for (int t = uni((int)(tid >> 6)); t < tokens; t += 4) {
    int64_t s, nth;
    const Seq q = seq_of_slot(d.batch, d.cache.page, 1, 0, 0, t0 + t, &s, &nth, err);
    int64_t pos = (int64_t)q.n_kv - q.n_new + nth;
    if (nth < 0 || nth >= q.n_new || pos < 0 || pos >= q.n_held) {
      pos = -1;
    } else if (d.pos) {
      pos = rope_pos(d, t0 + t);
      if (pos < 0) *err = OUT_OF_RANGE, pos = 0;
    }
    if ((tid & 63) == 0) place[t] = pos;
  }
  __syncthreads();
  for (int i = tid; i < tokens * half; i += 256) {
    const int t = i / half;
    if (place[t] >= 0) rope_angle(Angles{d.freq, d.amplitude, false}, place[t], i - t * half, &cs[i], &sn[i]);
  }
  __syncthreads();
  const bool tail = d.q.ptr != d.q_out.ptr;
  const int units = pairs + (tail ? (columns - rot + 2 * V - 1) / (2 * V) : 0);
  const int wide = units < 256 ? units : 256, step = 256 / wide, stride = step * g.parts, total = tokens * heads;
  if (tid >= wide * step) return;
  for (int u = tid % wide; u < units; u += wide) {
    int a, b;
    rope_columns<INTER, V>(u, pairs, half, rot, &a, &b);
    const bool two = b < columns;
    if (!two) b = a;
    int row = block % g.parts * step + tid / wide, t = 0, h = row;
    while (row < total) {
      RopeRaw<DT, V> r[R];
      int at[R];
      int64_t to[R];
      bool on[R];
#pragma unroll
      for (int k = 0; k < R; ++k) {
        while (h >= heads) {
          h -= heads;
          ++t;
        }
        on[k] = row < total && place[t < tokens ? t : 0] >= 0;
        to[k] = (t0 + t) * d.q_out.tok + h * d.q_out.head;
        at[k] = t * half + u * V;
        if (on[k]) {
          const int64_t e = (t0 + t) * d.q.tok + h * d.q.head;
          rope_load<DT, V, PAST>(d.q.ptr, e + a, e + b, r[k]);
        }
        row += stride;
        h += stride;
      }
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (!on[k]) continue;
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
        rope_store<DT, V>(d.q_out.ptr, to[k] + a, to[k] + b, r[k], two);
      }
    }
  }
}

// ---- keys and values ------------------------------------------------------------

template <int DT>
__device__ __forceinline__ float of16(const New16& x, int i) {
  const uint32_t w = x.w[i >> 1];
  if constexpr (DT == KTIR_BF16) return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w >> 16 : w));
}

// 16 columns from `col` on of a row at element e, turned by the angles of its row at cs, sn
template <int DT, bool INTER>
__device__ __forceinline__ void turned16(const ktir_kv8_rope_append_t& d, uint64_t ptr, int64_t e, int col, bool wide, bool vectors, const float* cs, const float* sn, float* x) {
  const int half = (int)d.rot / 2, rot = (int)d.rot;
  const New16 own = new16(ptr, e + col, wide);
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = of16<DT>(own, i);
  if (col >= rot) return;
  if constexpr (INTER) {
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      if (col + i >= rot) break;
      const float c = cs[(col + i) / 2], s = sn[(col + i) / 2], a = x[i], b = x[i + 1];
      x[i] = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
      x[i + 1] = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
    }
  } else if (vectors) {                        // half a multiple of 8: eight columns have their partners side by side
#pragma unroll
    for (int v = 0; v < 16; v += 8) {
      const int c0 = col + v;
      if (c0 >= rot) break;
      const bool first = c0 < half;
      const int at = first ? c0 : c0 - half;
      const u4_t w = *((const KTIR_G(u4_t)*)(ptr + 2 * (e + (first ? c0 + half : c0 - half))));
      const New16 other = {{w.x, w.y, w.z, w.w, 0, 0, 0, 0}};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = of16<DT>(other, i), t = __fmul_rn(p, sn[at + i]), y = __fmul_rn(x[v + i], cs[at + i]);
        x[v + i] = first ? __fsub_rn(y, t) : __fadd_rn(y, t);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int c0 = col + i;
      if (c0 >= rot) break;
      const bool first = c0 < half;
      const int at = first ? c0 : c0 - half;
      const float p = load_elem(ptr, e + (first ? c0 + half : c0 - half), DT), t = __fmul_rn(p, sn[at]), y = __fmul_rn(x[i], cs[at]);
      x[i] = first ? __fsub_rn(y, t) : __fadd_rn(y, t);
    }
  }
}

__device__ __forceinline__ u4_t codes_of16(const float* x, float f, int code) {
  u4_t o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float v[4] = {x[4 * i] * f, x[4 * i + 1] * f, x[4 * i + 2] * f, x[4 * i + 3] * f};
    o[i] = code == KTIR_I8 ? codes4<KTIR_I8>(v) : codes4<KTIR_E4M3>(v);
  }
  return o;
}

// W wavefronts have a page's part of a head (of K: IS_K, else of V).
template <int DT, bool INTER, int W, bool IS_K>
__device__ __forceinline__ void turn_kv(const ktir_kv8_rope_append_t& d, int slot, int group, float* cs, float* sn, uint32_t* tops, int* err) {
  const ktir_kv8_t& c = d.cache;
  const int wave = uni((int)(threadIdx.x >> 6)), tid = W == 1 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
  const int64_t head = W == 1 ? group * 4 + wave : group;
  int64_t s, nth;
  const int shift = __builtin_ctz((uint32_t)c.page);
  const Seq q = seq_of_slot(d.batch, c.page, 1, shift, 2, slot, &s, &nth, err);
  if (nth < 0) return;
  const int64_t pos0 = (int64_t)q.n_kv - q.n_new, from = pos0 < 0 ? 0 : pos0;      // the first position that is stored
  const int64_t p = (from >> shift) + nth;                                       // the page's number in the sequence
  const int64_t lo = p << shift < from ? from : p << shift, hi = (p + 1) << shift < q.n_held ? (p + 1) << shift : q.n_held;
  if (lo >= hi) return;
  const int64_t at = ints(d.batch.table)[s * d.batch.table_row + p];
  const int n = (int)(hi - lo), r0 = (int)(lo & (c.page - 1)), half = (int)d.rot / 2;
  const int64_t t0 = q.start + lo - pos0;
  const ktir_rows3_t& in = IS_K ? d.k : d.v;
  const int G = (int)c.columns >> 4, per = 64 * W / G, r = tid / G, col = (tid - r * G) * 16;     // rows a pass; this thread's
  const bool wide = !((in.ptr | (uint64_t)in.tok * 2 | (uint64_t)in.head * 2) & 15), mine = r < per && head < c.heads;
  const int64_t e0 = t0 * in.tok + head * in.head;

  // the angles of the rows from `first` on, as many as there are up to `most`
  auto angles = [&](int first, int most) {
    const int rows = n - first < most ? n - first : most;
    for (int i = threadIdx.x; i < rows * half; i += 256) {
      const int row = i / half;
      int64_t pos = d.pos ? rope_pos(d, t0 + first + row) : lo + first + row;
      if (pos < 0) *err = OUT_OF_RANGE, pos = 0;
      rope_angle(Angles{d.freq, d.amplitude, false}, pos, i - row * half, &cs[i], &sn[i]);
    }
  };
  // row `row`'s columns, its angles those of row `of` in LDS
  auto load = [&](int row, int of, float* x) {
    if constexpr (IS_K) {
      turned16<DT, INTER>(d, in.ptr, e0 + row * in.tok, col, wide, wide && half % 8 == 0, cs + of * half, sn + of * half, x);
    } else {
      const New16 own = new16(in.ptr, e0 + row * in.tok + col, wide);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = of16<DT>(own, i);
    }
  };
  // absolute bits: they grow with the value, and past infinity's for NaN
  auto most_of = [&](const float* x, uint32_t top) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t b = __float_as_uint(x[i]) & 0x7fffffffu;
      top = top > b ? top : b;
    }
    return top;
  };
  float x[TURN_KEPT][16];
  uint32_t top = 0;
  if constexpr (W == 1) {                    // a page has TURN_KEPT passes of rows at most: all its angles at once
    if constexpr (IS_K) {
      angles(0, n);
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < TURN_KEPT; ++i)
      if (mine && i * per + r < n) load(i * per + r, i * per + r, x[i]);
#pragma unroll
    for (int i = 0; i < TURN_KEPT; ++i)
      if (mine && i * per + r < n) top = most_of(x[i], top);
  } else {
#pragma unroll
    for (int i = 0; i < TURN_KEPT; ++i) {
      if (i * per >= n) break;
      if constexpr (IS_K) {
        __syncthreads();
        angles(i * per, per);
        __syncthreads();
      }
      if (mine && i * per + r < n) {
        load(i * per + r, r, x[i]);
        top = most_of(x[i], top);
      }
    }
    for (int row = TURN_KEPT * per; row < n; row += per) {
      float y[16];
      if constexpr (IS_K) {
        __syncthreads();
        angles(row, per);
        __syncthreads();
      }
      if (mine && row + r < n) {
        load(row + r, r, y);
        top = most_of(y, top);
      }
    }
  }
  if (at < 0 || at >= c.pages) {
    *err = OUT_OF_RANGE;
    return;
  }
  KTIR_G(uint8_t)* codes = (KTIR_G(uint8_t)*)(IS_K ? c.k + at * c.k_page + head * c.k_head : c.v + at * c.v_page + head * c.v_head) + col;
  const int64_t tok = IS_K ? c.k_tok : c.v_tok;
  KTIR_G(float)* scale = IS_K ? (KTIR_G(float)*)c.k_scale + at * c.ks_page + head * c.ks_head
                              : (KTIR_G(float)*)c.v_scale + at * c.vs_page + head * c.vs_head;
  const float before = r0 && head < c.heads ? *scale : 0.f;
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
  const float most = __uint_as_float(top), per_top = c.dtype == KTIR_I8 ? PER_TOP<KTIR_I8> : PER_TOP<KTIR_E4M3>;
  float now = __builtin_fmaxf(most * per_top, LEAST_SCALE);
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
        if (c.dtype == KTIR_I8) values4<KTIR_I8>(y[i], v);
        else values4<KTIR_E4M3>(y[i], v);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] *= ratio;
        y[i] = c.dtype == KTIR_I8 ? codes4<KTIR_I8>(v) : codes4<KTIR_E4M3, true>(v);
      }
      *w = y;
    }
  }
  const u4_t none = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < TURN_KEPT; ++i)
    if (mine && i * per + r < n) *(KTIR_G(u4_t)*)(codes + (r0 + i * per + r) * tok) = nan ? none : codes_of16(x[i], inv, c.dtype);
  if constexpr (W > 1) {
    for (int row = TURN_KEPT * per; row < n; row += per) {
      float y[16];
      if constexpr (IS_K) {
        __syncthreads();
        angles(row, per);
        __syncthreads();
      }
      if (mine && row + r < n) {
        load(row + r, r, y);
        *(KTIR_G(u4_t)*)(codes + (r0 + row + r) * tok) = nan ? none : codes_of16(y, inv, c.dtype);
      }
    }
  }
  if (tid == 0 && head < c.heads) *scale = now;
}

template <int DT, bool INTER, int V, bool PAST, int W>
__global__ __launch_bounds__(256) void kv8_turn(const ktir_kv8_rope_append_t d, const TurnGrid g, int* err) {
  __shared__ __attribute__((aligned(16))) float cs[TURN_PAIRS], sn[TURN_PAIRS];
  __shared__ int64_t place[TURN_TOKENS];
  __shared__ uint32_t tops[4];
  const int block = blockIdx.x, kv = 2 * g.kv * g.slots;
  if (block >= kv) return turn_queries<DT, INTER, V, PAST>(d, block - kv, g, cs, sn, place, err);
  const int slot = block / (2 * g.kv), group = block - slot * 2 * g.kv;
  if (group < g.kv) turn_kv<DT, INTER, W, true>(d, slot, group, cs, sn, tops, err);
  else turn_kv<DT, INTER, W, false>(d, slot, group - g.kv, cs, sn, tops, err);
}

// whether every vector of 8 values of the queries starts on a 16-byte bound
static bool wide_rows(const ktir_rows3_t& r, int64_t tokens, int64_t heads) {
  return !(r.ptr & 15) && (tokens == 1 || r.tok % 8 == 0) && (heads == 1 || r.head % 8 == 0);
}

template <int DT, bool INTER, int W>
static int turn_go(const ktir_kv8_rope_append_t& d, hipStream_t st) {
  constexpr const char* ME = "ktir_launch_kv8_rope_append";
  const int64_t tokens = d.batch.tokens, half = d.rot / 2, columns = d.cache.columns;
  const bool wide = half % 8 == 0 && (columns - d.rot) % 8 == 0 && wide_rows(d.q, tokens, d.q_heads) && wide_rows(d.q_out, tokens, d.q_heads);
  const int V = wide ? 8 : 1;
  TurnGrid g;
  // a sequence's n new tokens touch at most floor(n / page) + 2 pages
  const int64_t slots = tokens / d.cache.page + 2 * d.batch.seqs;
  g.kv = (int)(W == 1 ? (d.cache.heads + 3) / 4 : d.cache.heads);
  // the queries: as ktir_rope.hip cuts them
  const int64_t units = half / V + (columns - d.rot + 2 * V - 1) / (2 * V), step = 256 / (units < 256 ? units : 256);
  int64_t per = tokens / 1024;
  per = per > TURN_TOKENS ? TURN_TOKENS : per < 1 ? 1 : per;
  if (per * half > TURN_PAIRS) per = TURN_PAIRS / half;
  const int64_t blocks = (tokens + per - 1) / per;
  int64_t parts = 1;
  if (blocks < 512) {
    parts = (per * d.q_heads + step - 1) / step;
    const int64_t most = (1024 + blocks - 1) / blocks;
    parts = parts > most ? most : parts;
  }
  if (2 * g.kv * slots + blocks * parts > INT32_MAX) return set_error(KTIR_E_UNSUPPORTED, "%s: %lld pages, %lld heads in one launch", ME, (long long)slots, (long long)d.cache.heads);
  g.slots = (int)slots;
  g.per = (int)per;
  g.parts = (int)parts;
  const dim3 grid((unsigned)(2 * g.kv * slots + blocks * parts));
  const bool past = wide && d.q.ptr != d.q_out.ptr && 2 * tokens * d.q_heads * columns * 2 > (int64_t)64 << 20;      // (as ktir_rope.hip has it)
  if (past) hipLaunchKernelGGL((kv8_turn<DT, INTER, 8, true, W>), grid, dim3(256), 0, st, d, g, device_error_flag());
  else if (wide) hipLaunchKernelGGL((kv8_turn<DT, INTER, 8, false, W>), grid, dim3(256), 0, st, d, g, device_error_flag());
  else hipLaunchKernelGGL((kv8_turn<DT, INTER, 1, false, W>), grid, dim3(256), 0, st, d, g, device_error_flag());
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}

template <int DT>
static int turn_type(const ktir_kv8_rope_append_t& d, hipStream_t st) {
  // a page's units fit into one wavefront's registers: four heads share a workgroup
  if (d.cache.page * (d.cache.columns / 16) <= 64 * TURN_KEPT) return d.interleaved ? turn_go<DT, true, 1>(d, st) : turn_go<DT, false, 1>(d, st);
  return d.interleaved ? turn_go<DT, true, 4>(d, st) : turn_go<DT, false, 4>(d, st);
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
  const hipStream_t st = stream_of(d->stream);
  return d->dtype == KTIR_BF16 ? turn_type<KTIR_BF16>(*d, st) : turn_type<KTIR_F16>(*d, st);
}
