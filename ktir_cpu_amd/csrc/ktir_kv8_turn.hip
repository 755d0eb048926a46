// Rotary positions and append to the 8-bit cache in one launch.
//
// Two kinds of workgroups.  One turns queries: a few tokens, whose angles it makes once (in 64
// bits) for all heads, two rows of 16-byte loads a thread ahead of the stores.  The other has a page that new
// tokens fall in, and K or V: one, two or four wavefronts a head, its turned values in f32 registers from the maximum to the
// codes.  A unit of K loads its 16 columns and those that they are turned with, which a neighbour
// has just loaded: all layouts of pairs then store 16 codes at once.
//
// Bound: bytes, queries in and out and keys and values in once, codes out.  8192 tokens of 32 / 8 heads of 128 columns, 185
// MB: 43.6 us = 4.2 TB/s in a loop of launches, 45.6 (44.7 to 47.3) in a card's first ones (a copy of 256 MiB makes 5.4; the rotation and the
// append by themselves take 31.8 and 12.5).  On a card where it takes 40.8: 182 us with an element a thread, 52 with four units a thread (fewer wavefronts a CU), 47.6 with the loads behind the
// angles, 43 with eight tokens a workgroup of queries.  The two kinds in turn take 63 to 70: in one launch their
// streams do not go together.  Queries first 44.4, four rows of loads ahead 43.7.
// Few tokens are latency, and have kernels of their own below.
#include <type_traits>

#include "ktir_kv8_codes.h"
#include "ktir_rope_dev.h"

namespace ktir {

constexpr int TURN_TOKENS = 8;       // of a workgroup that turns queries
constexpr int TURN_KEPT = 2;         // units of 16 columns that a thread keeps
// angles in LDS: eight tokens' queries, or the keys of the rows that W wavefronts keep (64 W units each, half of 16 columns a unit)
constexpr int turn_pairs(int W) { return 1024 * W; }

// how a launch is cut: workgroups of keys and values first, then those of queries
struct TurnGrid {
  int kv, slots;       // workgroups for a page, of keys, then as many of values; pages
  int per, parts;      // tokens of a workgroup of queries, workgroups that share their heads
};

__device__ __forceinline__ double frequency(const ktir_kv8_rope_append_t& d, int i) { return ((const KTIR_G(double)*)d.freq)[i]; }
// The angles of `rows` rows into cs and sn, by all threads; `first`: the frequency of a thread's first
// pair, loaded before anything else is known; pos(row): a row's position, below 0 for one without
template <class Pos>
__device__ __forceinline__ void turn_angles(const ktir_kv8_rope_append_t& d, int rows, double first, float* cs, float* sn, Pos pos) {
  const int half = (int)d.rot / 2, total = rows * half;
  const bool same = 256 % half == 0;                 // a thread's pairs are one
  double f = first;
  for (int i = threadIdx.x; i < total;) {
    const int row = i / half;
    const int64_t p = pos(row);
    if (p >= 0) rope_angle_of(p, f, d.amplitude, false, &cs[i], &sn[i]);
    i += 256;
    if (!same && i < total) f = frequency(d, i % half);
  }
}

// The position of a token's rotation; false where the token is not stored.
__device__ __forceinline__ bool token_position(const ktir_kv8_rope_append_t& d, int64_t token, int64_t* pos, int* err) {
  int64_t s, nth;
  const int64_t given = d.pos ? rope_pos(d, token) : 0;
  const Seq q = seq_of_slot(d.batch, d.cache.page, 1, 0, 0, token, &s, &nth, err);
  const int64_t place = (int64_t)q.n_kv - q.n_new + nth;
  if (nth < 0 || nth >= q.n_new || place < 0 || place >= q.n_held) return false;
  if (given < 0) *err = OUT_OF_RANGE;
  *pos = !d.pos ? place : given < 0 ? 0 : given;
  return true;
}

// What of a page's slot of a launch is new: n rows from row r0 on, tokens from t0 on, whose places are from lo on.
struct PagePart {
  int64_t page, t0, lo;
  int n, r0;
  bool there;          // whether the table's page is one of the cache's
};
// page number `p` of sequence s, which is q
__device__ __forceinline__ bool part_of(const ktir_kv8_rope_append_t& d, const Seq& q, int64_t s, int64_t p, PagePart* part) {
  const ktir_kv8_t& c = d.cache;
  const int shift = __builtin_ctz((uint32_t)c.page);
  const int64_t pos0 = (int64_t)q.n_kv - q.n_new, from = pos0 < 0 ? 0 : pos0;      // the first position that is stored
  const int64_t lo = p << shift < from ? from : p << shift, hi = (p + 1) << shift < q.n_held ? (p + 1) << shift : q.n_held;
  if (lo >= hi) return false;
  const int64_t page = ints(d.batch.table)[s * d.batch.table_row + p];
  *part = {page, q.start + lo - pos0, lo, (int)(hi - lo), (int)(lo & (c.page - 1)), page >= 0 && page < c.pages};
  return true;
}
__device__ __forceinline__ bool page_part(const ktir_kv8_rope_append_t& d, int slot, PagePart* part, int* err) {
  const int shift = __builtin_ctz((uint32_t)d.cache.page);
  int64_t s, nth;
  const Seq q = seq_of_slot(d.batch, d.cache.page, 1, shift, 2, slot, &s, &nth, err);
  if (nth < 0) return false;
  const int64_t pos0 = (int64_t)q.n_kv - q.n_new;
  return part_of(d, q, s, ((pos0 < 0 ? 0 : pos0) >> shift) + nth, part);
}
// Part `at` of those of more than `most` rows (fewer than a page has), of all sequences in order; false where there are not as
// many.  All lanes of a wavefront search together, 64 sequences a step.
__device__ __forceinline__ bool long_part(const ktir_kv8_rope_append_t& d, int64_t at, int most, PagePart* part, int* err) {
  const int64_t page = d.cache.page;
  const int l = threadIdx.x & 63, shift = __builtin_ctz((uint32_t)page);
  for (int64_t base = 0; base < d.batch.seqs; base += 64) {
    Seq q = {0, 0, 0, 0};
    if (base + l < d.batch.seqs) q = seq_of(d.batch, page, base + l, err);
    const int64_t from = q.n_kv > q.n_new ? q.n_kv - q.n_new : 0, end = q.n_held;
    const int64_t first = from >> shift, last = (end - 1) >> shift, head = ((first + 1) << shift < end ? (first + 1) << shift : end) - from;
    // (all pages between the first and the last are full)
    const int begins = head > most, n = end <= from ? 0 : first == last ? begins : begins + (int)(last - first - 1) + (end - (last << shift) > most);
    int upto = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(upto, o);
      upto += l >= o ? y : 0;
    }
    const uint64_t past = __ballot(at < upto);
    if (past) {
      const int i = __builtin_ctzll(past), nth = (int)at - (lane_of(upto, i) - lane_of(n, i));
      return part_of(d, lane_of(q, i), base + i, lane_of(first, i) + nth + 1 - lane_of(begins, i), part);
    }
    at -= lane_of(upto, 63);
  }
  return false;
}
__device__ __forceinline__ int64_t row_position(const ktir_kv8_rope_append_t& d, const PagePart& part, int row, int* err) {
  const int64_t pos = d.pos ? rope_pos(d, part.t0 + row) : part.lo + row;
  if (pos < 0) *err = OUT_OF_RANGE;
  return pos < 0 ? 0 : pos;
}

// Where a page's part of a head of K or V lies.
struct PageHead {
  KTIR_G(uint8_t)* codes;
  KTIR_G(float)* scale;
  int64_t tok;
  __device__ __forceinline__ PageHead(const ktir_kv8_rope_append_t& d, const PagePart& part, int64_t head, bool is_k) {
    const ktir_kv8_t& c = d.cache;
    codes = (KTIR_G(uint8_t)*)(is_k ? c.k + part.page * c.k_page + head * c.k_head : c.v + part.page * c.v_page + head * c.v_head);
    scale = is_k ? (KTIR_G(float)*)c.k_scale + part.page * c.ks_page + head * c.ks_head : (KTIR_G(float)*)c.v_scale + part.page * c.vs_page + head * c.vs_head;
    tok = is_k ? c.k_tok : c.v_tok;
  }
};

// A page's scale with new values, of absolute bits `top` at most (they grow with the value, and past infinity's for NaN).
struct NewScale {
  float scale, inv, ratio;
  bool nan;
  __device__ __forceinline__ NewScale(int code, uint32_t top, float before) {
    const float most = __uint_as_float(top);
    scale = __builtin_fmaxf(most * (code == KTIR_I8 ? PER_TOP<KTIR_I8> : PER_TOP<KTIR_E4M3>), LEAST_SCALE);
    if (!(scale >= before)) scale = before;                     // a page that was NaN stays so
    if (!(most < __builtin_inff())) scale = __builtin_nanf("");
    nan = !(scale < __builtin_inff());
    inv = 1.f / scale;
    ratio = before * inv;
  }
  // the page's older rows, up to `end`, rounded to it by `threads` threads
  __device__ __forceinline__ void again(const ktir_kv8_t& c, KTIR_G(uint8_t)* codes, int64_t tok, int end, int tid, int threads) const {
    const int G = (int)c.columns >> 4;
    for (int i = tid; i < end * G; i += threads) {
      KTIR_G(u4_t)* w = (KTIR_G(u4_t)*)(codes + i / G * tok + i % G * 16);
      u4_t y = *w;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float v[4];
        if (c.dtype == KTIR_I8) values4<KTIR_I8>(y[k], v);
        else values4<KTIR_E4M3>(y[k], v);
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] *= ratio;
        y[k] = c.dtype == KTIR_I8 ? codes4<KTIR_I8>(v) : codes4<KTIR_E4M3, true>(v);
      }
      *w = y;
    }
  }
};

// ---- queries -----------------------------------------------------------------

template <int DT, bool INTER, int V, bool PAST>
__device__ __forceinline__ void turn_queries(const ktir_kv8_rope_append_t& d, int block, const TurnGrid& g, float* cs, float* sn, int64_t* place, int* err) {
  constexpr int R = 2;
  const double f0 = frequency(d, threadIdx.x % (uint32_t)(d.rot / 2));
  const int tid = threadIdx.x, half = (int)d.rot / 2, rot = (int)d.rot, columns = (int)d.cache.columns, pairs = half / V;
  const int64_t t0 = (int64_t)(block / g.parts) * g.per;
  const int tokens = (int)(d.batch.tokens - t0 < g.per ? d.batch.tokens - t0 : g.per), heads = (int)d.q_heads;
  const bool tail = d.q.ptr != d.q_out.ptr;
  const int units = pairs + (tail ? (columns - rot + 2 * V - 1) / (2 * V) : 0);
  const int wide = units < 256 ? units : 256, step = 256 / wide, stride = step * g.parts, total = tokens * heads;
  // R rows of a unit at a time; the first ones' loads are ahead of the angles
  struct Rows {
    RopeRaw<DT, V> r[R];
    int t[R], h[R];
  };
  int u = tid % wide, a, b;
  bool two;
  auto columns_of = [&]() {
    rope_columns<INTER, V>(u, pairs, half, rot, &a, &b);
    two = b < columns;                       // the last unit behind rot may be half one
    if (!two) b = a;
  };
  auto fetch = [&](int row, Rows& x) {
#pragma unroll
    for (int k = 0; k < R; ++k, row += stride) {
      x.t[k] = (int)((uint32_t)row / (uint32_t)heads);
      x.h[k] = row - x.t[k] * heads;
      if (row < total) {
        const int64_t e = (t0 + x.t[k]) * d.q.tok + x.h[k] * d.q.head;
        rope_load<DT, V, PAST>(d.q.ptr, e + a, e + b, x.r[k]);
      } else {
        x.t[k] = -1;
      }
    }
  };
  const int row0 = block % g.parts * step + tid / wide;
  const bool mine = tid < wide * step;
  Rows now;
  columns_of();
  if (mine) fetch(row0, now);
  // a token's position, or -1 where it is not stored
  auto position = [&](int64_t token) {
    int64_t pos;
    return token_position(d, token, &pos, err) ? pos : (int64_t)-1;
  };
  int64_t one = -1;
  if (g.per == 1) {                          // every wavefront by itself: a barrier less
    one = position(t0);
    turn_angles(d, 1, f0, cs, sn, [&](int) { return one; });
  } else {
    for (int t = uni((int)(tid >> 6)); t < tokens; t += 4) {
      const int64_t pos = position(t0 + t);
      if ((tid & 63) == 0) place[t] = pos;
    }
    __syncthreads();
    turn_angles(d, tokens, f0, cs, sn, [&](int t) { return place[t]; });
  }
  __syncthreads();
  auto live = [&](int t) { return (g.per == 1 ? one : place[t]) >= 0; };
  if (!mine) return;
  for (;;) {
    for (int row = row0; row < total; row += R * stride) {
      if (row != row0) fetch(row, now);
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (now.t[k] < 0 || !live(now.t[k])) continue;
        if (u < pairs) {
          __attribute__((aligned(16))) float c[V], s[V];
          const int at = now.t[k] * half + u * V;
          if constexpr (V > 1) {                             // half and so every unit's angles: multiples of 4
#pragma unroll
            for (int i = 0; i < V; i += 4) {
              *(f4_t*)(c + i) = *(const f4_t*)&cs[at + i];
              *(f4_t*)(s + i) = *(const f4_t*)&sn[at + i];
            }
          } else {
            c[0] = cs[at];
            s[0] = sn[at];
          }
          rope_turn_raw<DT, INTER, V>(now.r[k], c, s);
        }
        const int64_t to = (t0 + now.t[k]) * d.q_out.tok + now.h[k] * d.q_out.head;
        rope_store<DT, V>(d.q_out.ptr, to + a, to + b, now.r[k], two);
      }
    }
    u += wide;
    if (u >= units) return;
    columns_of();
    fetch(row0, now);
  }
}

// ---- keys and values ------------------------------------------------------------

template <int DT>
__device__ __forceinline__ float of16(const New16& x, int i) {
  const uint32_t w = x.w[i >> 1];
  if constexpr (DT == KTIR_BF16) return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w >> 16 : w));
}

// 16 columns of a row, and those that they are turned with
struct Raw16 {
  New16 own, other;
};

// `vectors`: half is a multiple of 8, so eight columns have their partners side by side on a 16-byte bound
template <int DT, bool INTER>
__device__ __forceinline__ void load16(const ktir_kv8_rope_append_t& d, uint64_t ptr, int64_t e, int col, bool wide, bool vectors, Raw16& x) {
  const int half = (int)d.rot / 2, rot = (int)d.rot;
  x.own = new16(ptr, e + col, wide);
  if constexpr (!INTER) {
    auto partner = [&](int c0) { return e + (c0 < half ? c0 + half : c0 - half); };
#pragma unroll
    for (int v = 0; v < 16; v += 8) {
      if (col + v >= rot) break;
      if (vectors) {
        const u4_t w = *(const KTIR_G(u4_t)*)(ptr + 2 * partner(col + v));
#pragma unroll
        for (int i = 0; i < 4; ++i) x.other.w[v / 2 + i] = w[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t w = col + v + i < rot ? ((const KTIR_G(uint16_t)*)ptr)[partner(col + v + i)] : 0u;
          x.other.w[(v + i) / 2] = i & 1 ? x.other.w[(v + i) / 2] | w << 16 : w;
        }
      }
    }
  }
}

// turned by the angles of their row at cs, sn
template <int DT, bool INTER>
__device__ __forceinline__ void turn16(const ktir_kv8_rope_append_t& d, const Raw16& raw, int col, bool vectors, const float* cs, const float* sn, float* x) {
  const int half = (int)d.rot / 2, rot = (int)d.rot;
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = of16<DT>(raw.own, i);
  if constexpr (INTER) {
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      if (col + i >= rot) break;
      const float c = cs[(col + i) / 2], s = sn[(col + i) / 2], a = x[i], b = x[i + 1];
      x[i] = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
      x[i + 1] = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
    }
  } else {
#pragma unroll
    for (int v = 0; v < 16; v += 8) {
      if (col + v >= rot) break;
      __attribute__((aligned(16))) float c[8], s[8];
      if (vectors) {
        const int at = col + v < half ? col + v : col + v - half;
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          *(f4_t*)(c + i) = *(const f4_t*)&cs[at + i];
          *(f4_t*)(s + i) = *(const f4_t*)&sn[at + i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int c0 = col + v + i, at = c0 < half ? c0 : c0 < rot ? c0 - half : 0;
          c[i] = cs[at], s[i] = sn[at];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (col + v + i >= rot) break;
        const float t = __fmul_rn(of16<DT>(raw.other, v + i), s[i]), y = __fmul_rn(x[v + i], c[i]);
        x[v + i] = col + v + i < half ? __fsub_rn(y, t) : __fadd_rn(y, t);
      }
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

// W wavefronts have a page's part of a head (of K: IS_K, else of V); MORE: it may have rows past those that they keep.
template <int DT, bool INTER, int W, bool MORE, bool IS_K>
__device__ __forceinline__ void turn_kv(const ktir_kv8_rope_append_t& d, int slot, int group, float* cs, float* sn, uint32_t* tops, int* err) {
  const ktir_kv8_t& c = d.cache;
  const int wave = uni((int)(threadIdx.x >> 6)), tid = (int)threadIdx.x & (64 * W - 1);
  const int64_t head = group * (4 / W) + wave / W;
  const double f0 = IS_K ? frequency(d, threadIdx.x % (uint32_t)(d.rot / 2)) : 0.0;
  PagePart part;
  if (!page_part(d, slot, &part, err)) return;
  const int n = part.n, r0 = part.r0, half = (int)d.rot / 2;
  const ktir_rows3_t& in = IS_K ? d.k : d.v;
  const int G = (int)c.columns >> 4, per = 64 * W / G, r = tid / G, col = (tid - r * G) * 16;     // rows a pass; this thread's
  const bool wide = !((in.ptr | (uint64_t)in.tok * 2 | (uint64_t)in.head * 2) & 15), mine = r < per && head < c.heads;
  const int64_t e0 = part.t0 * in.tok + head * in.head;
  const PageHead to(d, part, head, IS_K);
  float before = 0.f;
  // the unit of 16 columns of the rows first + r, first + per + r, ...: loads, then (K) the angles of these rows into LDS, then the values
  const bool vectors = wide && half % 8 == 0;
  auto values = [&](int first, float (&x)[TURN_KEPT][16]) {
    Raw16 raw[TURN_KEPT];
#pragma unroll
    for (int i = 0; i < TURN_KEPT; ++i) {
      const int row = first + i * per + r;
      if (!mine || row >= n) continue;
      if constexpr (IS_K) load16<DT, INTER>(d, in.ptr, e0 + row * in.tok, col, wide, vectors, raw[i]);
      else raw[i].own = new16(in.ptr, e0 + row * in.tok + col, wide);
    }
    if (first == 0 && r0 && part.there && head < c.heads) before = *to.scale;
    if constexpr (IS_K) {
      if (first) __syncthreads();
      const int rows = n - first < TURN_KEPT * per ? n - first : TURN_KEPT * per;
      turn_angles(d, rows, f0, cs, sn, [&](int row) { return row_position(d, part, first + row, err); });
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < TURN_KEPT; ++i) {
      if (!mine || first + i * per + r >= n) continue;
      if constexpr (IS_K) {
        turn16<DT, INTER>(d, raw[i], col, vectors, cs + (i * per + r) * half, sn + (i * per + r) * half, x[i]);
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) x[i][k] = of16<DT>(raw[i].own, k);
      }
    }
  };
  uint32_t top = 0;
  auto look = [&](int first, const float (&x)[TURN_KEPT][16]) {
#pragma unroll
    for (int i = 0; i < TURN_KEPT; ++i) {
      if (!mine || first + i * per + r >= n) continue;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const uint32_t y = __float_as_uint(x[i][k]) & 0x7fffffffu;
        top = top > y ? top : y;
      }
    }
  };
  // rows past those that are kept are read again, from the cache
  float x[TURN_KEPT][16];
  values(0, x);
  look(0, x);
  if constexpr (MORE) {
#pragma unroll 1
    for (int first = TURN_KEPT * per; first < n; first += TURN_KEPT * per) {
      float y[TURN_KEPT][16];
      values(first, y);
      look(first, y);
    }
  }
  if (!part.there) {
    *err = OUT_OF_RANGE;
    return;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const uint32_t y = __shfl_xor(top, o);
    top = top > y ? top : y;
  }
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) tops[wave] = top;
    __syncthreads();                       // also: every wavefront has read the scale before it changes
#pragma unroll
    for (int i = 0; i < W; ++i) top = top > tops[wave / W * W + i] ? top : tops[wave / W * W + i];
  }
  const NewScale now(c.dtype, top, before);
  if (now.scale > before && r0 && head < c.heads) now.again(c, to.codes, to.tok, r0, tid, 64 * W);
  const u4_t none = {0, 0, 0, 0};
  auto store = [&](int first, const float (&x)[TURN_KEPT][16]) {
#pragma unroll
    for (int i = 0; i < TURN_KEPT; ++i) {
      const int row = first + i * per + r;
      if (mine && row < n) *(KTIR_G(u4_t)*)(to.codes + (r0 + row) * to.tok + col) = now.nan ? none : codes_of16(x[i], now.inv, c.dtype);
    }
  };
  store(0, x);
  if constexpr (MORE) {
#pragma unroll 1
    for (int first = TURN_KEPT * per; first < n; first += TURN_KEPT * per) {
      float y[TURN_KEPT][16];
      values(first, y);
      store(first, y);
    }
  }
  if (tid == 0 && head < c.heads) *to.scale = now.scale;
}

template <int DT, bool INTER, int V, bool PAST, int W, bool MORE>
__global__ __launch_bounds__(256, MORE ? 1 : 4) void kv8_turn(const ktir_kv8_rope_append_t d, const TurnGrid g, int* err) {
  __shared__ __attribute__((aligned(16))) float cs[turn_pairs(W)], sn[turn_pairs(W)];
  __shared__ int64_t place[TURN_TOKENS];
  __shared__ uint32_t tops[4];
  const int kv = 2 * g.kv * g.slots, block = blockIdx.x;
  if (block >= kv) return turn_queries<DT, INTER, V, PAST>(d, block - kv, g, cs, sn, place, err);
  const int slot = block / (2 * g.kv), group = block - slot * 2 * g.kv;
  if (group < g.kv) turn_kv<DT, INTER, W, MORE, true>(d, slot, group, cs, sn, tops, err);
  else turn_kv<DT, INTER, W, MORE, false>(d, slot, group - g.kv, cs, sn, tops, err);
}

// ---- few tokens ---------------------------------------------------------------------
//
// A decode step, or a few drafts of each sequence, is latency: the instructions of one wavefront, one after
// another, and its loads.  Here a lane has pairs of one row (and columns behind the turned ones), so an angle is made where
// it is used, without LDS, and what a wavefront does is short.  A workgroup has a page's part of a head of K or
// V, a row a wavefront (of four heads, a wavefront each, where most sequences have a token or two), or one token's part of
// the queries, a head a wavefront at a time.

constexpr int FEW_TOKENS = 8;
constexpr int FEW_HEADS = 16;        // of the queries, for a workgroup
constexpr int FEW_KEPT = 2;          // rows that a wavefront keeps
constexpr int FEW_WIDE = 256;        // workgroups for longer ones
static_assert(4 * FEW_KEPT >= FEW_TOKENS, "four wavefronts read no row again");

struct FewAngles {
  float c[2], s[2];                  // of pairs l and l + 64
};
struct FewRow {
  float pair[2][2], rest[4];         // columns rot + l + 64 i
};

__device__ __forceinline__ FewAngles few_angles(const ktir_kv8_rope_append_t& d, int64_t pos, const double (&f)[2]) {
  FewAngles a;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if ((int)(threadIdx.x & 63) + 64 * i < d.rot / 2) rope_angle_of(pos, f[i], d.amplitude, false, &a.c[i], &a.s[i]);
  return a;
}

// where the first column of a lane's pair i lies, and how far the second is from it
__device__ __forceinline__ int few_first(const ktir_kv8_rope_append_t& d, int i) {
  const int p = (threadIdx.x & 63) + 64 * i;
  return d.interleaved ? 2 * p : p;
}
__device__ __forceinline__ int few_gap(const ktir_kv8_rope_append_t& d) { return d.interleaved ? 1 : (int)d.rot / 2; }

// The same by a call, for a loop over rows: inline, the constants of sine and cosine stay in registers around the loop, which costs
// the short parts of the same kernel wavefronts (1024 sequences of one token 60.2 us, 57.8).
struct OneAngle {
  float c, s;
};
__device__ __attribute__((noinline)) OneAngle one_angle(int64_t pos, double freq, double amplitude) {
  OneAngle a;
  rope_angle_of(pos, freq, amplitude, false, &a.c, &a.s);
  return a;
}
__device__ __forceinline__ FewAngles few_angles_again(const ktir_kv8_rope_append_t& d, int64_t pos, const double (&f)[2]) {
  FewAngles a;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if ((int)(threadIdx.x & 63) + 64 * i < d.rot / 2) {
      const OneAngle x = one_angle(pos, f[i], d.amplitude);
      a.c[i] = x.c, a.s[i] = x.s;
    }
  return a;
}

template <int DT>
__device__ __forceinline__ void few_load(const ktir_kv8_rope_append_t& d, uint64_t ptr, int64_t e, bool rest, FewRow& x) {
  const int l = threadIdx.x & 63, half = (int)d.rot / 2;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (l + 64 * i < half) {
      x.pair[i][0] = load_elem(ptr, e + few_first(d, i), DT);
      x.pair[i][1] = load_elem(ptr, e + few_first(d, i) + few_gap(d), DT);
    }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (rest && d.rot + l + 64 * i < d.cache.columns) x.rest[i] = load_elem(ptr, e + d.rot + l + 64 * i, DT);
}

__device__ __forceinline__ void few_turn(FewRow& x, const FewAngles& a) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float u = x.pair[i][0], v = x.pair[i][1];
    x.pair[i][0] = __fsub_rn(__fmul_rn(u, a.c[i]), __fmul_rn(v, a.s[i]));
    x.pair[i][1] = __fadd_rn(__fmul_rn(v, a.c[i]), __fmul_rn(u, a.s[i]));
  }
}

template <int DT>
__device__ __forceinline__ void few_queries(const ktir_kv8_rope_append_t& d, int block, int parts, const double (&f)[2], int* err) {
  const int64_t token = block / parts;
  const int wave = uni((int)(threadIdx.x >> 6)), l = threadIdx.x & 63, half = (int)d.rot / 2;
  const int h0 = block % parts * FEW_HEADS, end = h0 + FEW_HEADS < d.q_heads ? h0 + FEW_HEADS : (int)d.q_heads;
  const bool rest = d.q.ptr != d.q_out.ptr;
  FewRow x;
  if (h0 + wave < end) few_load<DT>(d, d.q.ptr, token * d.q.tok + (h0 + wave) * d.q.head, rest, x);
  int64_t pos;
  if (!token_position(d, token, &pos, err)) return;
  const FewAngles a = few_angles(d, pos, f);
  for (int h = h0 + wave; h < end; h += 4) {
    if (h != h0 + wave) few_load<DT>(d, d.q.ptr, token * d.q.tok + h * d.q.head, rest, x);
    few_turn(x, a);
    const int64_t e = token * d.q_out.tok + h * d.q_out.head;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (l + 64 * i < half) {
        store_elem(d.q_out.ptr, e + few_first(d, i), DT, x.pair[i][0]);
        store_elem(d.q_out.ptr, e + few_first(d, i) + few_gap(d), DT, x.pair[i][1]);
      }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (rest && d.rot + l + 64 * i < d.cache.columns) store_elem(d.q_out.ptr, e + d.rot + l + 64 * i, DT, x.rest[i]);
  }
}

// W wavefronts (1 or 4) have a page's part of a head, a row each in turn: rows that they keep between the maximum and
// the codes, or (MORE) any number, each read twice.
template <int DT, int W, bool MORE>
__device__ __forceinline__ void few_kv(const ktir_kv8_rope_append_t& d, const PagePart& part, int64_t head, bool is_k, const double (&f)[2], uint32_t* tops, int* err) {
  const ktir_kv8_t& c = d.cache;
  const int wave = W == 1 ? 0 : uni((int)(threadIdx.x >> 6)), l = threadIdx.x & 63, half = (int)d.rot / 2;
  const ktir_rows3_t in = is_k ? d.k : d.v;
  const int64_t e0 = part.t0 * in.tok + head * in.head;
  auto values = [&](int row, FewRow& x) {
    few_load<DT>(d, in.ptr, e0 + row * in.tok, true, x);
    if (!is_k) return;
    const int64_t pos = row_position(d, part, row, err);
    few_turn(x, MORE ? few_angles_again(d, pos, f) : few_angles(d, pos, f));
  };
  uint32_t top = 0;
  auto look = [&](const FewRow& x) {
    auto see = [&](float v) {
      const uint32_t y = __float_as_uint(v) & 0x7fffffffu;
      top = top > y ? top : y;
    };
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (l + 64 * i < half) see(x.pair[i][0]), see(x.pair[i][1]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d.rot + l + 64 * i < c.columns) see(x.rest[i]);
  };
  FewRow x[FEW_KEPT];                      // (MORE: unused)
  const PageHead to(d, part, head, is_k);
  const float before = part.there && part.r0 ? *to.scale : 0.f;
  if constexpr (MORE) {
#pragma unroll 1
    for (int row = wave; row < part.n; row += W) {
      values(row, x[0]);
      look(x[0]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < FEW_KEPT; ++k)
      if (wave + W * k < part.n) {
        values(wave + W * k, x[k]);
        look(x[k]);
      }
  }
  if (!part.there) {
    *err = OUT_OF_RANGE;
    return;
  }
  for (int o = 32; o; o >>= 1) {
    const uint32_t y = __shfl_xor(top, o);
    top = top > y ? top : y;
  }
  if constexpr (W > 1) {
    if (l == 0) tops[wave] = top;
    __syncthreads();                       // also: every wavefront has read the scale before it changes
#pragma unroll
    for (int i = 0; i < W; ++i) top = top > tops[i] ? top : tops[i];
  }
  const NewScale now(c.dtype, top, before);
  if (now.scale > before && part.r0) now.again(c, to.codes, to.tok, part.r0, 64 * wave + l, 64 * W);
  auto put = [&](int row, const FewRow& x) {
    KTIR_G(uint8_t)* p = to.codes + (part.r0 + row) * to.tok;
    float a[4] = {x.pair[0][0] * now.inv, x.pair[0][1] * now.inv, x.pair[1][0] * now.inv, x.pair[1][1] * now.inv};
    float b[4] = {x.rest[0] * now.inv, x.rest[1] * now.inv, x.rest[2] * now.inv, x.rest[3] * now.inv};
    uint32_t u = c.dtype == KTIR_I8 ? codes4<KTIR_I8>(a) : codes4<KTIR_E4M3>(a), v = c.dtype == KTIR_I8 ? codes4<KTIR_I8>(b) : codes4<KTIR_E4M3>(b);
    if (now.nan) u = v = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (l + 64 * i < half) {
        p[few_first(d, i)] = (uint8_t)(u >> (16 * i));
        p[few_first(d, i) + few_gap(d)] = (uint8_t)(u >> (16 * i + 8));
      }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d.rot + l + 64 * i < c.columns) p[d.rot + l + 64 * i] = (uint8_t)(v >> (8 * i));
  };
  if constexpr (MORE) {
#pragma unroll 1
    for (int row = wave; row < part.n; row += W) {
      values(row, x[0]);
      put(row, x[0]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < FEW_KEPT; ++k)
      if (wave + W * k < part.n) put(wave + W * k, x[k]);
  }
  if (wave == 0 && l == 0) *to.scale = now.scale;
}

// `wide` workgroups come first, for parts that are too long for one wavefront: a batch of a token or two a sequence may have
// most of them in one, which the host does not know.  Each looks for its parts itself and ends where there are no more.  256
// sequences of one token and one of 200, pages of 16, 64 and 256: 17.3, 34.2 and 58.8 us (28.8, 83.8 and 163.8 with a wavefront for each part,
// 18.6, 50.9 and 112 in the other kernel); what they cost where there are no long parts: 64 of one token 6.1 -> 6.5, 256 11.6 -> 12.7.
template <int DT, int W>
__global__ __launch_bounds__(256) void kv8_turn_few(const ktir_kv8_rope_append_t d, int slots, int groups, int parts, int wide, int* err) {
  __shared__ uint32_t tops[4];
  const int l = threadIdx.x & 63, half = (int)d.rot / 2, heads = (int)d.cache.heads, kv = groups * slots, block = (int)blockIdx.x - wide;
  const double f[2] = {frequency(d, l < half ? l : 0), frequency(d, l + 64 < half ? l + 64 : 0)};
  if (block >= kv) return few_queries<DT>(d, block - kv, parts, f, err);
  PagePart part;
  if (W == 1 && block < 0) {
    // (the descriptor by an address that the compiler does not know: else it is loaded, and spilled, before the branch; 64 of one token 7.4 us)
    auto* again = (const __attribute__((address_space(4))) ktir_kv8_rope_append_t*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(again));
    const ktir_kv8_rope_append_t& d = *(const ktir_kv8_rope_append_t*)again;
    for (int64_t at = blockIdx.x;; at += wide) {
      const int64_t nth = at / (2 * heads);
      const int hv = (int)(at - nth * 2 * heads);
      if (!long_part(d, nth, FEW_KEPT, &part, err)) return;
      few_kv<DT, 4, true>(d, part, hv < heads ? hv : hv - heads, hv < heads, f, tops, err);
      __syncthreads();
    }
  }
  const int slot = block / groups, hv = (block - slot * groups) * (4 / W) + (W == 1 ? uni((int)(threadIdx.x >> 6)) : 0);
  if (hv >= 2 * heads || !page_part(d, slot, &part, err) || (W == 1 && part.n > FEW_KEPT)) return;
  if (hv < heads) few_kv<DT, W, false>(d, part, hv, true, f, tops, err);
  else few_kv<DT, W, false>(d, part, hv - heads, false, f, tops, err);
}

// whether every vector of 8 values of the queries starts on a 16-byte bound
static bool wide_rows(const ktir_rows3_t& r, int64_t tokens, int64_t heads) {
  return !(r.ptr & 15) && (tokens == 1 || r.tok % 8 == 0) && (heads == 1 || r.head % 8 == 0);
}

template <int DT, bool INTER, int W, bool MORE>
static int turn_go(const ktir_kv8_rope_append_t& d, hipStream_t st) {
  constexpr const char* ME = "ktir_launch_kv8_rope_append";
  const int64_t tokens = d.batch.tokens, half = d.rot / 2, columns = d.cache.columns;
  const bool wide = half % 8 == 0 && (columns - d.rot) % 8 == 0 && wide_rows(d.q, tokens, d.q_heads) && wide_rows(d.q_out, tokens, d.q_heads);
  const int V = wide ? 8 : 1;
  TurnGrid g;
  // a sequence's n new tokens touch at most floor(n / page) + 2 pages
  const int64_t slots = tokens / d.cache.page + 2 * d.batch.seqs;
  g.kv = (int)((d.cache.heads + 4 / W - 1) / (4 / W));
  // the queries: as ktir_rope.hip cuts them
  const int64_t units = half / V + (columns - d.rot + 2 * V - 1) / (2 * V), step = 256 / (units < 256 ? units : 256);
  int64_t per = tokens / 2048;
  per = per > TURN_TOKENS ? TURN_TOKENS : per < 1 ? 1 : per;
  const int64_t blocks = (tokens + per - 1) / per;
  int64_t parts = 1;
  if (blocks < 512) {
    parts = (per * d.q_heads + step - 1) / step;
    const int64_t most = (1024 + blocks - 1) / blocks;
    parts = parts > most ? most : parts;
  }
  const int64_t kv = 2 * g.kv * slots, queries = blocks * parts;
  if (kv > (1 << 29) || queries > (1 << 29)) return set_error(KTIR_E_UNSUPPORTED, "%s: %lld pages, %lld heads in one launch", ME, (long long)slots, (long long)d.cache.heads);
  g.slots = (int)slots;
  g.per = (int)per;
  g.parts = (int)parts;
  const dim3 grid((unsigned)(kv + queries));
  const bool past = wide && d.q.ptr != d.q_out.ptr && 2 * tokens * d.q_heads * columns * 2 > (int64_t)64 << 20;      // (as ktir_rope.hip has it)
  if (past) hipLaunchKernelGGL((kv8_turn<DT, INTER, 8, true, W, MORE>), grid, dim3(256), 0, st, d, g, device_error_flag());
  else if (wide) hipLaunchKernelGGL((kv8_turn<DT, INTER, 8, false, W, MORE>), grid, dim3(256), 0, st, d, g, device_error_flag());
  else hipLaunchKernelGGL((kv8_turn<DT, INTER, 1, false, W, MORE>), grid, dim3(256), 0, st, d, g, device_error_flag());
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}

template <int DT>
static int turn_type(const ktir_kv8_rope_append_t& d, hipStream_t st) {
  // The kernels for few tokens, four wavefronts a head for up to 8 (32 / 8 heads of 128 columns, one sequence of 1 to 4: 4.6 us,
  // of 8 5.5, the other kernel 6.6 to 7.0; 16 in pages of 64 8.4 and 7.2), one where there are up to two a sequence on average (64
  // sequences of one 6.5, of two 7.4, the other kernel 7.5 and 7.7, with pages of 64 6.5 and 12.8; 256 of one 12.5 and 15.9) and four
  // for a part of more (64 of one and 40 of another sequence, pages of 16 and 64, 12.7 and 21.3, the other kernel 10.4 and 18.2).
  const bool few = d.batch.tokens <= FEW_TOKENS;
  if (few || d.batch.tokens <= 2 * d.batch.seqs) {
    const int64_t slots = d.batch.tokens / d.cache.page + 2 * d.batch.seqs, parts = (d.q_heads + FEW_HEADS - 1) / FEW_HEADS;
    const int64_t groups = few ? 2 * d.cache.heads : (2 * d.cache.heads + 3) / 4, most = d.batch.tokens / (FEW_KEPT + 1) * 2 * d.cache.heads;
    const int64_t wide = few ? 0 : most < FEW_WIDE ? most : FEW_WIDE, blocks = wide + groups * slots + d.batch.tokens * parts;
    if (blocks <= (1 << 30)) {
      if (!few) hipLaunchKernelGGL((kv8_turn_few<DT, 1>), dim3((unsigned)blocks), dim3(256), 0, st, d, (int)slots, (int)groups, (int)parts, (int)wide, device_error_flag());
      else hipLaunchKernelGGL((kv8_turn_few<DT, 4>), dim3((unsigned)blocks), dim3(256), 0, st, d, (int)slots, (int)groups, (int)parts, 0, device_error_flag());
      KTIR_HIP_CHECK(hipGetLastError());
      return KTIR_OK;
    }
  }
  // a page's units fit into the registers of one wavefront, or of two: several heads share a workgroup (and their angles).
  // (64 W / G rows a pass, two passes: whole pages of 16 rows or more for all G up to 8 W)
  const int64_t G = d.cache.columns / 16, units = d.cache.page * G;
  const bool whole = TURN_KEPT * (256 / G) >= d.cache.page;
  auto go = [&](auto inter) {
    constexpr bool INTER = decltype(inter)::value;
    return units <= 128 ? turn_go<DT, INTER, 1, false>(d, st) : units <= 256 ? turn_go<DT, INTER, 2, false>(d, st)
                     : whole ? turn_go<DT, INTER, 4, false>(d, st) : turn_go<DT, INTER, 4, true>(d, st);
  };
  return d.interleaved ? go(std::true_type()) : go(std::false_type());
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
