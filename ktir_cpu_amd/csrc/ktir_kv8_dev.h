// Device helpers of the attention kernels over an 8-bit cache.
//
// Keys' codes become f16 operands, which hold both code types exactly, and so do
// queries of either type, each row times a power of two; so every product of a
// score is exact (but for elements below 2^-28 of a bf16 row's largest) and their
// sum is the matrix instruction's f32.
//
// The scales stay out of the operands: with t_j = log2(e) scale kscale q . k_j and
// page scales kscale, vscale,
//   w_j = 2^(t_j + log2 vscale - b) = vscale p_j 2^-b   enters the product with V's codes,
//   l = 2^-16 sum w_j / vscale,  out = 2^-16 (sum w_j code_j) / l,  lse = (b + 16 + log2 l) ln 2,
// one addition per page and one multiply-add per weight (2^-16 keeps l finite
// for 2^28 keys whose vscale is the least, 2^-100).  b follows the row's largest exponent.
#pragma once
#include "ktir_attn_common.h"
#include "ktir_serve.h"

namespace ktir {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x3_t __attribute__((ext_vector_type(3), aligned(4)));

constexpr float B_LAG = 8.f;                     // b is changed when an exponent passes it by more
constexpr float B_NONE = -1e38f;                 // b of a row that has seen no key
constexpr float L_UNIT = 0x1p-16f;
constexpr float LEAST_V = 0x1p-100f;             // the least vscale that w is computed with (append's least; smaller ones count as this)

template <bool BF16>
__device__ __forceinline__ f32x4_t mfma16(const uint4& a, const uint4& b, f32x4_t c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

// bytes `lo` of x and `hi` of y as the low bytes of two halves, zeros above
template <int LO, int HI>
__device__ __forceinline__ uint32_t bytes2(uint32_t x, uint32_t y) {
  return __builtin_amdgcn_perm(y, x, 0x0c000c00u | (uint32_t)(4 + HI) << 16 | (uint32_t)LO);
}

// such a pair of i8 codes as f16: 0x6400 + (c + 128) is 1152 + c
__device__ __forceinline__ uint32_t i8_half2(uint32_t w) {
  const f16x2_t v = __builtin_bit_cast(f16x2_t, w ^ 0x64806480u), off = {(_Float16)-1152.f, (_Float16)-1152.f};
  return __builtin_bit_cast(uint32_t, v + off);
}

// codes 2 k, 2 k + 1 of a word
template <int CODE, int K>
__device__ __forceinline__ uint32_t word_half2(uint32_t w) {
  if constexpr (CODE == KTIR_I8) return i8_half2(bytes2<2 * K, 2 * K + 1>(w, w));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, K == 1));
}

// eight codes in a row
template <int CODE>
__device__ __forceinline__ uint4 row_half8(uint32_t w0, uint32_t w1) {
  return make_uint4(word_half2<CODE, 0>(w0), word_half2<CODE, 1>(w0), word_half2<CODE, 0>(w1), word_half2<CODE, 1>(w1));
}

// two words, four codes each, as four bf16 pairs (x's code, y's code)
template <int CODE>
__device__ __forceinline__ void cross_bf2(uint32_t x, uint32_t y, uint32_t (&out)[4]) {
  if constexpr (CODE == KTIR_I8) {
#pragma unroll
    for (int n = 0; n < 4; ++n) out[n] = cvt2<true>((float)(int8_t)(x >> (8 * n)), (float)(int8_t)(y >> (8 * n)));
  } else {
    const uint32_t a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false)),
                   b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, 1.0f, false)),
                   c = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true)),
                   e = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, 1.0f, true));
    out[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    out[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    out[2] = __builtin_amdgcn_perm(e, c, 0x05040100u);
    out[3] = __builtin_amdgcn_perm(e, c, 0x07060302u);
  }
}

// two words, four codes each, as four f16 pairs (x's code, y's code)
template <int CODE>
__device__ __forceinline__ void cross_half2(uint32_t x, uint32_t y, uint32_t (&out)[4]) {
  if constexpr (CODE == KTIR_I8) {
    out[0] = i8_half2(bytes2<0, 0>(x, y));
    out[1] = i8_half2(bytes2<1, 1>(x, y));
    out[2] = i8_half2(bytes2<2, 2>(x, y));
    out[3] = i8_half2(bytes2<3, 3>(x, y));
  } else {
    const uint32_t a = word_half2<CODE, 0>(x), b = word_half2<CODE, 0>(y), c = word_half2<CODE, 1>(x), e = word_half2<CODE, 1>(y);
    out[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    out[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    out[2] = __builtin_amdgcn_perm(e, c, 0x05040100u);
    out[3] = __builtin_amdgcn_perm(e, c, 0x07060302u);
  }
}

// Where the groups of 16 keys of a wavefront's next steps lie, a group per lane.
struct KV8Groups {
  int page;             // of the cache
  float ks, lv, iv;     // kscale, log2 vscale, 2^-16 / vscale
};

// The rows of one tile of a launch: query head h * grp + r % grp of token
// i = r / grp of sequence s, r from row0 on; what they see of the keys.
struct Tile {
  int64_t s;
  Seq q;
  int row0, rows;        // of the tile, rows 0: nothing to do
  int keys;              // cached tokens that count
  int lo, hi;            // tokens that some row of the tile sees
};

// tokens [lo, hi) that new token i of tile t's sequence sees
__device__ __forceinline__ void token_sees(const ktir_kv8_attn_t& d, const Tile& t, int i, int* lo, int* hi) {
  const int64_t pos = (int64_t)t.q.n_kv - t.q.n_new + i;
  *hi = d.causal && pos + 1 < t.keys ? (pos < 0 ? 0 : (int)(pos + 1)) : t.keys;
  *lo = d.window && pos - d.window + 1 > 0 ? (int)(pos - d.window + 1) : 0;
}
__device__ __forceinline__ void seen(const ktir_kv8_attn_t& d, const Tile& t, int r, int grp, int* lo, int* hi) {
  token_sees(d, t, (int)((uint32_t)r / (uint32_t)grp), lo, hi);
}

// tile `nth` (of TM rows) of sequence s, which is q
__device__ __forceinline__ Tile tile_at(const ktir_kv8_attn_t& d, int64_t s, const Seq& q, int64_t nth, int TM, int grp, int* err) {
  Tile t = {};
  t.s = s;
  t.q = q;
  t.keys = t.q.n_held;
  if (t.keys > d.max_k || t.q.n_new > d.max_q) *err = OUT_OF_RANGE;
  if (t.keys > d.max_k) t.keys = (int)d.max_k;
  const int64_t n = (t.q.n_new < d.max_q ? t.q.n_new : d.max_q) * grp, left = n - nth * TM;
  if (left <= 0) return t;
  t.row0 = (int)(nth * TM);
  t.rows = left < TM ? (int)left : TM;
  int x;
  if (nth == 0 && left <= TM) {              // the whole sequence: its first and last token
    token_sees(d, t, 0, &t.lo, &x);
    token_sees(d, t, (t.q.n_new < d.max_q ? t.q.n_new : (int)d.max_q) - 1, &x, &t.hi);
  } else {
    seen(d, t, t.row0, grp, &t.lo, &x);
    seen(d, t, t.row0 + t.rows - 1, grp, &x, &t.hi);
  }
  return t;
}

// whether a launch has one tile a sequence: its max_q tokens fit in TM (a power of two) rows
__host__ __device__ inline bool one_tile(const ktir_kv8_attn_t& d, int TM, int grp) { return d.max_q * grp <= TM; }

// tile `slot` of a launch: a sequence each, or found by the batch's offsets
__device__ __forceinline__ Tile tile_of(const ktir_kv8_attn_t& d, int64_t slot, int TM, int grp, int* err) {
  if (one_tile(d, TM, grp)) return tile_at(d, slot, seq_of(d.batch, d.cache.page, slot, err), 0, TM, grp, err);
  int64_t s, nth;
  const Seq q = seq_of_slot(d.batch, d.cache.page, grp, __builtin_ctz(TM), 1, slot, &s, &nth, err);
  return nth < 0 ? Tile{} : tile_at(d, s, q, nth, TM, grp, err);
}

// a tile's fields in scalar registers: they are the same in every lane, or lane i's
__device__ __forceinline__ Tile uni(Tile t) {
  t.s = uni(t.s);
  t.q.start = uni(t.q.start);
  t.q.n_new = uni(t.q.n_new);
  t.q.n_kv = uni(t.q.n_kv);
  t.row0 = uni(t.row0);
  t.rows = uni(t.rows);
  t.keys = uni(t.keys);
  t.lo = uni(t.lo);
  t.hi = uni(t.hi);
  return t;
}
__device__ __forceinline__ Tile lane_of(Tile t, int i) {
  t.s = lane_of(t.s, i);
  t.q.start = lane_of(t.q.start, i);
  t.q.n_new = lane_of(t.q.n_new, i);
  t.q.n_kv = lane_of(t.q.n_kv, i);
  t.row0 = lane_of(t.row0, i);
  t.rows = lane_of(t.rows, i);
  t.keys = lane_of(t.keys, i);
  t.lo = lane_of(t.lo, i);
  t.hi = lane_of(t.hi, i);
  return t;
}

// whether some row of the tile sees a key of the group that starts at `key`
__device__ __forceinline__ bool kv8_there(const Tile& t, int64_t key) { return key < t.hi && key + 16 > t.lo; }

// the page of the group that starts at `key`; of one that no row sees: page 0, which weighs
// nothing (before a window the table's entries may be those of pages that are gone)
__device__ __forceinline__ int kv8_pages(const ktir_kv8_attn_t& d, const Tile& t, int key, int shift) {
  return kv8_there(t, key) ? ints(d.batch.table)[t.s * d.batch.table_row + (key >> shift)] : 0;
}

__device__ __forceinline__ KV8Groups kv8_groups(const ktir_kv8_attn_t& d, int64_t head, int page, bool there, int* err) {
  if ((uint32_t)page >= (uint64_t)d.cache.pages) {
    *err = OUT_OF_RANGE;
    page = 0;
  }
  KV8Groups g = {page, 0.f, 0.f, L_UNIT};
  if (there) {
    g.ks = ((const KTIR_G(float)*)d.cache.k_scale)[page * d.cache.ks_page + head * d.cache.ks_head];
    g.lv = ((const KTIR_G(float)*)d.cache.v_scale)[page * d.cache.vs_page + head * d.cache.vs_head];
  }
  return g;
}

// vscale as its logarithm and inverse (not where it is loaded: that would wait for it)
__device__ __forceinline__ void kv8_scales(KV8Groups& g, bool there) {
  if (!there) return;
  const float vs = g.lv < LEAST_V ? LEAST_V : g.lv;
  g.lv = __builtin_amdgcn_logf(vs);
  g.iv = vs != vs ? 1.f : L_UNIT / vs;      // NaN is in lv, and so in the weights of the rows that see the page alone
}

// 16 query values from element e on, packed
__device__ __forceinline__ void q16(const ktir_kv8_attn_t& d, int64_t e, bool whole, uint32_t (&raw)[8]) {
  const KTIR_G(uint16_t)* p = (const KTIR_G(uint16_t)*)d.q.ptr + e;
  if (whole) {
    const u32x4_t a = ((const KTIR_G(u32x4_t)*)p)[0], b = ((const KTIR_G(u32x4_t)*)p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = a[i], raw[4 + i] = b[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) raw[i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
  }
}

// the largest of N packed pairs' absolute bits
template <int N>
__device__ __forceinline__ uint32_t top_bits(const uint32_t (&raw)[N], uint32_t top) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t a = raw[i] & 0x7fffu, b = (raw[i] >> 16) & 0x7fffu;
    top = top > a ? top : a;
    top = top > b ? top : b;
  }
  return top;
}

// f16 queries are operands as they are; bf16 ones take the power of two 2^k that brings the row's largest to 2^14
__device__ __forceinline__ int q_power(uint32_t top) {
  if (!top) return 0;
  const int k = 14 - ((int)(top >> 7) - 127);
  return k > 120 ? 120 : k < -113 ? -113 : k;
}
__device__ __forceinline__ float power2(int k) { return __uint_as_float((uint32_t)(127 + k) << 23); }

template <int N>
__device__ __forceinline__ void q_scaled(uint32_t (&raw)[N], float up) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const f32x2_t v = uncvt2<true>(raw[i]);
    raw[i] = cvt2<false>(v.x * up, v.y * up);
  }
}

}  // namespace ktir
