// Attention over the 8-bit cache for few rows: a decode step, a few speculative
// tokens, any launch that its keys must spread over the chip.
//
// A workgroup has a tile of 16 MT rows (tokens x the query heads of one KV head)
// and a range of the keys; `splits` workgroups share a tile's keys, and its
// four wavefronts share the workgroup's.  Each wavefront runs alone on its own
// keys, without barriers, 32 at a time:
//   S^T = K Q^T   16 x 16 x 32 MFMA: 16 keys x 16 rows, columns in the order that
//                 a lane's 16-byte load of a key's codes brings them (Q likewise)
//   w, b, l       as ktir_kv8_dev.h says; the maximum is looked at on every step,
//                 but changed, with O scaled, only where it grew by 2^8
//   O^T += V^T W^T  with V's codes in bf16, which holds them exactly, and w as two
//                 bf16 terms (17 bits of any weight, however small: one f16 term
//                 loses a key's where another of 2^25 times its weight has code 0);
//                 in the order of keys that the scores' layout leaves: no
//                 exchange between lanes; a lane's load of 4 J codes of eight
//                 keys is transposed by the byte selects of the conversion
// Pages, scales and addresses of 64 groups of 16 keys are fetched at once, one per
// lane, so no step waits for the chain table -> page -> key; K's codes of the next
// step are in flight while this one is computed (V's too: no faster, 35 registers more).
//
// Bound: bytes where the cache is long.  131072 tokens of 8 heads of 128, 269 MB of e4m3
// codes: 53.5 us = 5.0 TB/s and 4 to 7 us to join 128 parts; reads alone in this pattern
// make 5.6 TB/s.  More workgroups than two a CU lose DRAM locality (64 of 2460 tokens:
// 68.6 us with 512 workgroups, 81 with 1280).  Short ones are latency: one token after
// 1000 takes 7.0 us (launch, offsets -> table -> codes, two barriers) and 3.6 to join.
#include "ktir_kv8_dev.h"

namespace ktir {

constexpr int ROWS_WAVES = 4, ROWS_STEP = 32, ROWS_GROUPS = 64;
constexpr int MOST_SPLITS = 256;      // of a tile's keys

// what a split of a tile of `rows` rows leaves in the workspace: 64 J sums each, then b and l of each row
template <int J>
__host__ __device__ constexpr int64_t part_size(int rows) { return (int64_t)rows * (64 * J + 4); }

// the parts of a tile's keys, of `part` each
__device__ __forceinline__ int tile_parts(const Tile& t, int part) {
  const int from = t.lo & ~(ROWS_STEP - 1);
  return t.hi > from ? (int)((uint32_t)(t.hi - from + part - 1) / (uint32_t)part) : 1;
}

template <int J>
struct KV8Keys {
  u32x4_t k[2][J];
};
template <int J>
struct KV8Values {
  uint32_t v[8][J];
};

// the codes of 32 keys from `key` on; groups that the wavefront does not have read page 0
template <int J>
__device__ __forceinline__ void kv8_keys(const ktir_kv8_t& c, const KV8Groups& g, int group, int key, int64_t head, int koff,
                                         const int (&kpiece)[J], KV8Keys<J>& o) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t page = __builtin_amdgcn_readlane(g.page, group + h), row = (key + 16 * h) & (c.page - 1);
    const KTIR_G(uint8_t)* kp = (const KTIR_G(uint8_t)*)c.k + page * c.k_page + row * c.k_tok + head * c.k_head;
#pragma unroll
    for (int j = 0; j < J; ++j) o.k[h][j] = *(const KTIR_G(u32x4_t)*)(kp + (uint32_t)(koff + kpiece[j]));
  }
}

template <int J>
__device__ __forceinline__ void kv8_values(const ktir_kv8_t& c, const KV8Groups& g, int group, int key, int64_t head, int voff,
                                           KV8Values<J>& o) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t page = __builtin_amdgcn_readlane(g.page, group + h), row = (key + 16 * h) & (c.page - 1);
    const KTIR_G(uint8_t)* vp = (const KTIR_G(uint8_t)*)c.v + page * c.v_page + row * c.v_tok + head * c.v_head;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const KTIR_G(uint8_t)* p = vp + (uint32_t)(voff + i * (int)c.v_tok);
      if constexpr (J == 1) {
        o.v[4 * h + i][0] = *(const KTIR_G(uint32_t)*)p;
      } else if constexpr (J == 2) {
        const u32x2_t x = *(const KTIR_G(u32x2_t)*)p;
        o.v[4 * h + i][0] = x.x, o.v[4 * h + i][1] = x.y;
      } else if constexpr (J == 3) {
        const u32x3_t x = *(const KTIR_G(u32x3_t)*)p;
        o.v[4 * h + i][0] = x.x, o.v[4 * h + i][1] = x.y, o.v[4 * h + i][2] = x.z;
      } else {
        const u32x4_t x = *(const KTIR_G(u32x4_t)*)p;
#pragma unroll
        for (int j = 0; j < J; ++j) o.v[4 * h + i][j] = x[j];
      }
    }
  }
}

template <int CODE, int J, int MT>
__global__ __launch_bounds__(64 * ROWS_WAVES, MT == 1 ? 2 : 1) void kv8_attn_rows(const ktir_kv8_attn_t d, int splits, int part, int part_rows, uint32_t slots, int hw, int* err) {
  constexpr int W = ROWS_WAVES, TM = 16 * MT, N = 4 * J, PITCH = 64 * J + 4;
  __shared__ __attribute__((aligned(16))) float o_sum[W][TM * PITCH];
  __shared__ float w_b[W][TM], w_l[W][TM];
  const ktir_kv8_t& c = d.cache;
  const int l = threadIdx.x & 63, wave = uni((int)(threadIdx.x >> 6)), g4 = l >> 4, c16 = l & 15;
  const int grp = (int)((uint32_t)d.q_heads / (uint32_t)c.heads), D = (int)c.columns, shift = __builtin_ctz((uint32_t)c.page);
  // Workgroups go to the 8 XCDs in turn.  The heads of a part follow one another on one
  // XCD, so the rows of a page are read together; the parts that there are take the
  // XCDs in turn.
  const uint32_t heads = (uint32_t)c.heads, sets = heads / hw, octet = blockIdx.x / 8, eighth = octet / sets, u = eighth * 8 + blockIdx.x % 8;
  const int turn = wave / hw, TW = W / hw;                   // of the head's TW wavefronts
  const int64_t head = (octet - eighth * sets) * hw + wave % hw;
  Tile t;
  int split, active, from;
  uint32_t slot;
  if (d.batch.seqs == 1 && one_tile(d, TM, grp)) {
    slot = 0;
    split = (int)u;
    t = uni(tile_at(d, 0, seq_of(d.batch, c.page, 0, err), 0, TM, grp, err));
    if (!t.rows) return;
    active = tile_parts(t, part);
    if (split >= active) return;
  } else if (one_tile(d, TM, grp)) {
    // one tile a sequence, of as many parts as its keys fill: the u-th part of all, 64 sequences a look
    t.rows = 0;
    uint32_t before = 0;
    for (int64_t base = 0; base < d.batch.seqs; base += 64) {
      Tile x = {};
      if (base + l < d.batch.seqs) x = tile_at(d, base + l, seq_of(d.batch, c.page, base + l, err), 0, TM, grp, err);
      int n = x.rows ? tile_parts(x, part) : 0;
      n = n < splits ? n : splits;
      int upto = n;                                          // parts of the sequences up to this lane's
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(upto, o);
        upto += l >= o ? y : 0;
      }
      const uint32_t all = (uint32_t)lane_of(upto, 63);
      if (u < before + all) {
        const int i = __builtin_ctzll(__ballot(u < before + (uint32_t)upto));
        t = lane_of(x, i);
        active = lane_of(n, i);
        split = (int)(u - before) - (lane_of(upto, i) - active);
        slot = (uint32_t)base + i;
        break;
      }
      before += all;
    }
    if (!t.rows) return;
  } else {
    split = (int)(u / slots);
    slot = u - split * slots;
    if (split >= splits) return;
    t = uni(tile_of(d, slot, TM, grp, err));
    if (!t.rows) return;
    active = tile_parts(t, part);
    if (split >= active) return;
  }
  from = t.lo & ~(ROWS_STEP - 1);
  const int64_t item = (int64_t)slot * heads + head;
  // (steps of 32 keys go to the splits' wavefronts in turn, so what all read at one time lies close together)
  const int stride = ROWS_STEP * TW * active, lo = from + (split * TW + turn) * ROWS_STEP, mine = (l >> 1) * stride + 16 * (l & 1);
  const int page0 = kv8_pages(d, t, lo + mine, shift);

  // Q: this lane's row of each 16, pieces g4 J .. g4 J + J of 16 columns (so a load of K touches whole 128-byte lines); times 2^k, so that the row's largest value has exponent 14
  uint4 qf[MT][J][2];
  float rs[MT];
  int see_lo[MT], see_hi[MT], kpiece[J];
  uint32_t raw[MT][J][8];
#pragma unroll
  for (int j = 0; j < J; ++j) kpiece[j] = (g4 * J + j) * 16 < D ? (g4 * J + j) * 16 : 0;
  const bool whole = !((d.q.ptr | (uint64_t)d.q.tok * 2 | (uint64_t)d.q.head * 2) & 15);
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    int r = t.row0 + 16 * m + c16;
    if (r >= t.row0 + t.rows) r = t.row0 + t.rows - 1;              // a row that is not stored
    seen(d, t, r, grp, &see_lo[m], &see_hi[m]);
    const int64_t e = (t.q.start + r / grp) * d.q.tok + (head * grp + r % grp) * d.q.head;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int x = (g4 * J + j) * 16;
#pragma unroll
      for (int i = 0; i < 8; ++i) raw[m][j][i] = 0;
      if (x < D) q16(d, e + x, whole, raw[m][j]);
    }
  }
  const int koff = c16 * (int)c.k_tok, vcol = c16 * 4 * J + 4 * J <= D ? c16 * 4 * J : 0, voff = 4 * g4 * (int)c.v_tok + vcol;
  // the first keys' pages, scales and codes are on their way while Q is made ready
  KV8Groups g = kv8_groups(d, head, page0, kv8_there(t, lo + mine), err);
  KV8Keys<J> k[2];
  if (lo < t.hi) kv8_keys<J>(c, g, 0, lo, head, koff, kpiece, k[0]);
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) top = top_bits(raw[m][j], top);
    uint32_t y = __shfl_xor(top, 16);
    top = top > y ? top : y;
    y = __shfl_xor(top, 32);
    top = top > y ? top : y;
    const int up = d.dtype == KTIR_BF16 ? q_power(top) : 0;
    rs[m] = power2(-up) * (d.scale * LOG2E);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (d.dtype == KTIR_BF16) q_scaled(raw[m][j], power2(up));
      qf[m][j][0] = make_uint4(raw[m][j][0], raw[m][j][1], raw[m][j][2], raw[m][j][3]);
      qf[m][j][1] = make_uint4(raw[m][j][4], raw[m][j][5], raw[m][j][6], raw[m][j][7]);
    }
  }
  int lo_most, hi_least, x;
  seen(d, t, t.row0, grp, &x, &hi_least);
  seen(d, t, t.row0 + t.rows - 1, grp, &lo_most, &x);
  lo_most = uni(lo_most);
  hi_least = uni(hi_least);

  f32x4_t acc[MT][N];
  float b[MT], sum[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    b[m] = B_NONE;
    sum[m] = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n) acc[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  auto step = [&](const KV8Keys<J>& o, KV8Values<J>& ov, const KV8Groups& g, int group, int key) {
    f32x4_t s[MT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int m = 0; m < MT; ++m) s[m][h] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const uint4 a0 = row_half8<CODE>(o.k[h][j].x, o.k[h][j].y), a1 = row_half8<CODE>(o.k[h][j].z, o.k[h][j].w);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          s[m][h] = mfma16<false>(a0, qf[m][j][0], s[m][h]);
          s[m][h] = mfma16<false>(a1, qf[m][j][1], s[m][h]);
        }
      }
    }
    const bool cut = key < lo_most || key + ROWS_STEP > hi_least;
    const float ks[2] = {lane_of(g.ks, group), lane_of(g.ks, group + 1)}, lv[2] = {lane_of(g.lv, group), lane_of(g.lv, group + 1)},
                iv[2] = {lane_of(g.iv, group), lane_of(g.iv, group + 1)};
    uint4 wh[MT], wl[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      // exponents of the weights; a key that the row does not see has none
      float u[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float f = ks[h] * rs[m];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[4 * h + i] = __builtin_fmaf(s[m][h][i], f, lv[h]);
      }
      if (cut) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int j = key + 16 * (i >> 2) + 4 * g4 + (i & 3);
          u[i] = j < see_lo[m] || j >= see_hi[m] ? -__builtin_inff() : u[i];
        }
      }
      float top = u[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = __builtin_fmaxf(top, u[i]);
      if (__any(top > b[m] + B_LAG)) {
        top = __builtin_fmaxf(top, __shfl_xor(top, 16));
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        const float now = __builtin_fmaxf(b[m], top), keep = __builtin_amdgcn_exp2f(b[m] - now);
        b[m] = now;
        sum[m] *= keep;
#pragma unroll
        for (int n = 0; n < N; ++n) acc[m][n] *= keep;
      }
      uint32_t hi[4], lo_[4];
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float a = __builtin_amdgcn_exp2f(u[i] - b[m]), e = __builtin_amdgcn_exp2f(u[i + 1] - b[m]);
        sum[m] = __builtin_fmaf(a, iv[i >> 2], sum[m]);
        sum[m] = __builtin_fmaf(e, iv[i >> 2], sum[m]);
        hi[i / 2] = cvt2<true>(a, e);
        const f32x2_t back = uncvt2<true>(hi[i / 2]);
        lo_[i / 2] = cvt2<true>(a - back.x, e - back.y);
      }
      wh[m] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      wl[m] = make_uint4(lo_[0], lo_[1], lo_[2], lo_[3]);
    }
    if (CODE == KTIR_E4M3 && (key < t.lo || key + ROWS_STEP > t.hi)) {     // NaN codes of tokens that no row sees
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = key + 16 * (i >> 2) + 4 * g4 + (i & 3);
#pragma unroll
        for (int j = 0; j < J; ++j) ov.v[i][j] = at < t.lo || at >= t.hi ? 0u : ov.v[i][j];
      }
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      uint32_t p[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) cross_bf2<CODE>(ov.v[2 * i][j], ov.v[2 * i + 1][j], p[i]);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const uint4 a = make_uint4(p[0][n], p[1][n], p[2][n], p[3][n]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          acc[m][4 * j + n] = mfma16<true>(a, wl[m], acc[m][4 * j + n]);
          acc[m][4 * j + n] = mfma16<true>(a, wh[m], acc[m][4 * j + n]);
        }
      }
    }
  };

  for (int64_t first = lo; first < t.hi; first += (int64_t)stride * (ROWS_GROUPS / 2)) {
    const int base = (int)first;
    const bool there = kv8_there(t, first + mine);
    if (base != lo) {
      g = kv8_groups(d, head, there ? kv8_pages(d, t, base + mine, shift) : 0, there, err);
      kv8_keys<J>(c, g, 0, base, head, koff, kpiece, k[0]);
    }
    const int n = (t.hi - base + stride - 1) / stride, steps = n < ROWS_GROUPS / 2 ? n : ROWS_GROUPS / 2;
    for (int i = 0; i < steps; i += 2) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (i + x >= steps) break;
        const int key = base + stride * (i + x), group = 2 * (i + x);
        KV8Values<J> v;
        kv8_values<J>(c, g, group, key, head, voff, v);
        if (i + x + 1 < steps) kv8_keys<J>(c, g, group + 2, key + stride, head, koff, kpiece, k[1 - x]);
        if (x == 0 && i == 0) kv8_scales(g, there);      // with the first codes already on their way
        step(k[x], v, g, group, key);
      }
    }
  }

  // the wavefronts' sums, each in a part of LDS, then added in their order
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    sum[m] += __shfl_xor(sum[m], 16);
    sum[m] += __shfl_xor(sum[m], 32);
    if (g4 == 0) {
      w_b[wave][16 * m + c16] = b[m];
      w_l[wave][16 * m + c16] = sum[m];
    }
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int row = 16 * m + c16;
    float top = b[m];
    for (int w = wave % hw; w < W; w += hw) top = __builtin_fmaxf(top, w_b[w][row]);
    const float f = __builtin_amdgcn_exp2f(b[m] - top);
    if (row < t.rows) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < N; n += 4)
          *(f32x4_t*)(o_sum[wave] + row * PITCH + (4 * g4 + i) * N + n) =
              f32x4_t{acc[m][n][i] * f, acc[m][n + 1][i] * f, acc[m][n + 2][i] * f, acc[m][n + 3][i] * f};
    }
  }
  __syncthreads();

  // alone: the result; otherwise its part for kv8_attn_join
  KTIR_G(float)* ws = (KTIR_G(float)*)d.ws + (item * splits + split) * part_size<J>(part_rows);
  for (int at = turn * 64 + l; at < t.rows * 16 * J; at += 64 * TW) {
    const int row = at / (16 * J), x4 = at % (16 * J) * 4;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    float top = B_NONE, lt = 0.f;
    for (int w = wave % hw; w < W; w += hw) {
      o += *(const f32x4_t*)(o_sum[w] + row * PITCH + x4);
      top = __builtin_fmaxf(top, w_b[w][row]);
    }
    for (int w = wave % hw; w < W; w += hw) lt += w_l[w][row] * __builtin_amdgcn_exp2f(w_b[w][row] - top);
    if (active > 1) {
      *(KTIR_G(f32x4_t)*)(ws + row * 64 * J + x4) = o;
      if (x4 == 0) {
        ws[part_rows * 64 * J + row] = top;
        ws[part_rows * (64 * J + 1) + row] = lt;
      }
      continue;
    }
    const int r = t.row0 + row;
    int a, z;
    seen(d, t, r, grp, &a, &z);
    const int64_t tok = t.q.start + r / grp, h = head * grp + r % grp, e = tok * d.out.tok + h * d.out.head + x4;
    const float inv = L_UNIT / lt;
    if (x4 < D) {
#pragma unroll
      for (int i = 0; i < 4; ++i) store_elem(d.out.ptr, e + i, d.dtype, a >= z ? 0.f : o[i] * inv);
    }
    if (d.lse && x4 == 0)
      ((KTIR_G(float)*)d.lse)[tok * d.lse_tok + h * d.lse_head] =
          a >= z ? -__builtin_inff() : (top + 16.f + __builtin_amdgcn_logf(lt)) * 0.69314718055994530942f;
  }
}

// The parts of a tile's splits, joined: B wavefronts for each of R rows, which take
// up to 16 splits each in turn, J columns a lane.  Bound: latency.  All parts are
// read at once, before the sequence's length says which of them were written.
constexpr int JOIN_EACH = 16;

template <int J, int MT, int R, int B>
__global__ __launch_bounds__(64 * R * B) void kv8_attn_join(const ktir_kv8_attn_t d, int splits, int part, int part_rows, int* err) {
  constexpr int TM = 16 * MT, LOOK = B == 1 ? 1 : MOST_SPLITS / 64;
  static_assert(B * JOIN_EACH <= 64 * LOOK, "a lane looks at the b and l of each split");
  __shared__ float f[R][64 * LOOK], sums[B == 1 ? 1 : R * B][64 * J];
  const ktir_kv8_t& c = d.cache;
  const int l = threadIdx.x & 63, wave = uni((int)(threadIdx.x >> 6)), grp = (int)((uint32_t)d.q_heads / (uint32_t)c.heads), D = (int)c.columns;
  const uint32_t heads = (uint32_t)c.heads, slot = blockIdx.x / heads;
  const int64_t item = blockIdx.x, head = blockIdx.x - slot * heads;
  const int sub = wave / B, turn = wave % B, row = (int)blockIdx.y * R + sub;
  const int64_t size = part_size<J>(part_rows);
  const KTIR_G(float)* ws = (const KTIR_G(float)*)d.ws + item * splits * size;
  float x[JOIN_EACH][J], b[LOOK], w[LOOK];
#pragma unroll
  for (int i = 0; i < LOOK; ++i) {
    b[i] = B_NONE, w[i] = 0.f;
    if (row < part_rows && l + 64 * i < splits) {
      b[i] = ws[(l + 64 * i) * size + part_rows * 64 * J + row];
      w[i] = ws[(l + 64 * i) * size + part_rows * (64 * J + 1) + row];
    }
  }
#pragma unroll
  for (int k = 0; k < JOIN_EACH; ++k)
    if (row < part_rows && turn + B * k < splits) {
#pragma unroll
      for (int j = 0; j < J; ++j) x[k][j] = ws[(turn + B * k) * size + row * 64 * J + 64 * j + l];
    }
  const Tile t = uni(tile_of(d, slot, TM, grp, err));
  const int parts = tile_parts(t, part), active = parts < splits ? parts : splits;
  const bool on = row < t.rows && active > 1;
  float top = B_NONE, lt = 0.f;
#pragma unroll
  for (int i = 0; i < LOOK; ++i)
    if (l + 64 * i < active) top = __builtin_fmaxf(top, b[i]);
  for (int o = 32; o; o >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o));
#pragma unroll
  for (int i = 0; i < LOOK; ++i) {
    if (l + 64 * i >= active) continue;
    const float e = __builtin_amdgcn_exp2f(b[i] - top);
    lt += w[i] * e;
    if (turn == 0) f[sub][l + 64 * i] = e;
  }
  for (int o = 32; o; o >>= 1) lt += __shfl_xor(lt, o);
  __syncthreads();
  float acc[J] = {};
  if (on) {
#pragma unroll
    for (int k = 0; k < JOIN_EACH; ++k)
      if (turn + B * k < active) {
#pragma unroll
        for (int j = 0; j < J; ++j) acc[j] += x[k][j] * f[sub][turn + B * k];
      }
  }
  if constexpr (B > 1) {
#pragma unroll
    for (int j = 0; j < J; ++j) sums[wave][64 * j + l] = acc[j];
    __syncthreads();
    if (turn == 0) {
#pragma unroll
      for (int i = 1; i < B; ++i)
#pragma unroll
        for (int j = 0; j < J; ++j) acc[j] += sums[wave + i][64 * j + l];
    }
  }
  if (!on || turn) return;
  const int r = t.row0 + row;
  int a, z;
  seen(d, t, r, grp, &a, &z);
  const int64_t tok = t.q.start + r / grp, h = head * grp + r % grp;
  const float inv = L_UNIT / lt;
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (64 * j + l < D) store_elem(d.out.ptr, tok * d.out.tok + h * d.out.head + 64 * j + l, d.dtype, a >= z ? 0.f : acc[j] * inv);
  if (d.lse && l == 0)
    ((KTIR_G(float)*)d.lse)[tok * d.lse_tok + h * d.lse_head] =
        a >= z ? -__builtin_inff() : (top + 16.f + __builtin_amdgcn_logf(lt)) * 0.69314718055994530942f;
}

// the launch's shape: columns in 64s (192 alone has its three: other heads' loads of 12 codes would pass their end), rows, splits
void kv8_rows_shape(const ktir_kv8_attn_t& d, KV8Shape* s) {
  const int D = (int)d.cache.columns;
  const int64_t grp = d.q_heads / d.cache.heads;
  s->J = D <= 64 ? 1 : D <= 128 ? 2 : D == 192 ? 3 : 4;
  s->MT = d.max_q * grp > 16 ? 2 : 1;
  const int64_t TM = 16 * s->MT;
  s->slots = d.max_q * grp > TM ? d.batch.tokens * grp / TM + d.batch.seqs : d.batch.seqs;
  s->rows = (int)(d.max_q * grp < TM ? d.max_q * grp : TM);
  if (s->rows < 1) s->rows = 1;
  s->part = s->rows * (64 * s->J + 4);
  // the most tokens that a tile's rows see, from a step's bound on
  s->span = d.max_k;
  const int64_t near = d.window + (TM - 1) / grp + 1;
  if (d.window && near < s->span) s->span = near;
  s->span += ROWS_STEP - 1;
  // Heads of a workgroup, parts of the keys.  Up to 2^19 keys (times KV heads) a wavefront's
  // four work on one head, on parts of 128 keys or more: one workgroup a CU is best for one
  // sequence (65536 tokens of 8 heads: 36.8 us, two a CU 42.5), four for several (8 of up
  // to 8192: 20.5, 28.6 with one).  More come from HBM, which gives 4.8 TB/s to 128-byte
  // rows of one head each, 5.6 where four heads' rows are read together (read patterns of
  // 268 MB; 64 sequences of 2460 tokens: 77 and 68.6 us).  There one workgroup a CU is
  // best for one sequence (131072 tokens: 59.5 us, two 62.6); several, whose lengths the
  // host does not know, get four if all were the longest, with parts of 512 keys or more
  // (64 of 64 to 8192 tokens: parts of 1056 keys 78 us, of 832 74, of 2080 100, of 416 95;
  // 64 of 2460: parts of 640 68 us, of 256 81; 256 of up to 2048: of 544 88, of 1056 94).
  const int64_t heads = d.cache.heads, longest = s->span - (ROWS_STEP - 1), keys = s->slots * heads * longest;
  const bool tiles = !one_tile(d, (int)TM, (int)grp), far = keys > (1 << 19) && !tiles;
  s->HW = !far ? 1 : heads % 4 == 0 ? 4 : heads % 2 == 0 ? 2 : 1;
  const int64_t sets = s->slots * heads / s->HW;
  int64_t n = sets ? (tiles || s->slots <= 1 ? 256 : 1024) / sets : 1;
  if (far && s->slots > 1) {
    const int64_t even = longest / 512;
    n = n < 4 ? 4 : n;
    n = n < even ? n : even;
  }
  const int64_t most = (s->span + 127) / 128;
  n = n > most ? most : n;
  s->splits = n < 1 ? 1 : n > MOST_SPLITS ? MOST_SPLITS : (int)n;
}

template <int CODE, int J, int MT>
static int launch(const ktir_kv8_attn_t& d, const KV8Shape& s) {
  constexpr int W = ROWS_WAVES;
  const int64_t QUANT = ROWS_STEP * W / s.HW, items = s.slots * d.cache.heads, splits = d.splits < 1 ? 1 : d.splits;
  const int part = (int)(((s.span + splits - 1) / splits + QUANT - 1) / QUANT * QUANT);
  // two workgroups a CU, evenly: where three fit, some CUs get three and others one (510 parts of 704 keys: 89 and 72 us)
  constexpr int held = (int)(sizeof(float) * W * (16 * MT * (64 * J + 4) + 2 * 16 * MT)), spare = held < 55000 ? 55000 - held : 0;
  const hipStream_t st = stream_of(d.stream);
  hipLaunchKernelGGL((kv8_attn_rows<CODE, J, MT>), dim3((unsigned)((s.slots * splits + 7) / 8 * 8 * (d.cache.heads / s.HW))), dim3(64 * W), spare, st, d, (int)splits, part, s.rows, (uint32_t)s.slots, s.HW, device_error_flag());
  if (splits > 1) {
    if (splits <= JOIN_EACH) hipLaunchKernelGGL((kv8_attn_join<J, MT, 4, 1>), dim3((unsigned)items, (unsigned)((s.rows + 3) / 4)), dim3(256), 0, st, d, (int)splits, part, s.rows, device_error_flag());
    else hipLaunchKernelGGL((kv8_attn_join<J, MT, 1, 16>), dim3((unsigned)items, (unsigned)s.rows), dim3(1024), 0, st, d, (int)splits, part, s.rows, device_error_flag());
  }
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}

template <int CODE, int J>
static int launch_j(const ktir_kv8_attn_t& d, const KV8Shape& s) {
  return s.MT == 2 ? launch<CODE, J, 2>(d, s) : launch<CODE, J, 1>(d, s);
}

template <int CODE>
static int launch_code(const ktir_kv8_attn_t& d, const KV8Shape& s) {
  switch (s.J) {
    case 1: return launch_j<CODE, 1>(d, s);
    case 2: return launch_j<CODE, 2>(d, s);
    case 3: return launch_j<CODE, 3>(d, s);
    default: return launch_j<CODE, 4>(d, s);
  }
}

int kv8_rows_launch(const ktir_kv8_attn_t& d, const KV8Shape& s) {
  return d.cache.dtype == KTIR_I8 ? launch_code<KTIR_I8>(d, s) : launch_code<KTIR_E4M3>(d, s);
}

}  // namespace ktir
