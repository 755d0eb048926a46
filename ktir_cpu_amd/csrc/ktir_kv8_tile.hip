// Attention over the 8-bit cache for many rows: prompts and chunks of them.
//
// A workgroup has 256 rows (128 for more than 128 columns; tokens x the query heads of
// one KV head) of one sequence, 32 in each wavefront, and runs over the keys that they
// see, 64 at a time.  The codes of a step are made f16 once for all rows and laid into
// LDS (two buffers): K as [key][column], V as [column][key], with the keys of each 16 in
// the order that the scores' layout leaves them in:
//   S^T = K Q^T     32 x 32 x 16 MFMA, one row a lane (the two halves share it)
//   w, b, l         as ktir_kv8_dev.h says; w enters the product as two f16 terms
//   O^T += V^T W^T  no exchange between lanes
// With 65 to 128 columns the two wavefronts of a SIMD take turns, half a step apart: one
// makes the weights of its step (vector instructions alone), the other multiplies (the
// scores of its next step and W V of this one) and converts the codes of the step after;
// a barrier ends each half.  Else scores, conversion, weights and W V stand side by side,
// a quarter of each at a time: 64 columns 398 us so and 422 in turns, below.  A wavefront
// alone on its SIMD (more than 128 columns) has no one to take turns with.
//
// Bound: the instructions of a wavefront one after another, vector and matrix ones.  8192
// tokens, 32 / 8 heads of 128 columns, causal, i8 codes, 550 GFLOP and half as many for the
// second terms: 743 to 818 us on five cards (e4m3 739 to 781); 64 columns 504 to 525, 16 / 4 heads of
// 256 columns 1087 to 1098.  The matrix pipe is busy 51 % of the time, the vector pipe 58 %, LDS 30 %: the two
// wavefronts of a SIMD hardly cover each other.  A wavefront issues 41 % of its time and waits
// for data and barriers 32 %, for a pipe 27 %.  With one term of w 628 to 634, 598 to 605, 410 and 963 on the
// card of 815, the matrix pipe busy 44 %.
// Before, with one term: 1193 us in ktir_kv8_rows.hip, 906 with four wavefronts of 64 rows, 677 without the
// next scores beside, 630 side by side (634 on a card that takes 592 in turns); not faster: matrix instructions pinned
// between vector ones, seven to one (660 to 700), operands read six products ahead (604).  With two
// terms side by side takes 905 (e4m3 797), where turns take 778 (747).
//
// Two f16 terms, the weight rounded and what that leaves of it rounded again: w is at most 2^15, so
// down to 2^-3 a weight keeps 22 bits, and below that what is left is held in steps of
// 2^-24, which is 2^-35 to 2^-39 of the row's heaviest.  One term keeps 11 bits, which f16 results show.
#include <type_traits>

#include "ktir_kv8_dev.h"

namespace ktir {

constexpr int TILE_KEYS = 64;
constexpr float TILE_TOP = 11.f, TILE_LAG = 4.f;       // exponent of the largest weight when b changes, and by how much it may grow

// Slots of 16-byte chunks in LDS rows: a K row has 8 J (8 columns each), a V column 8 (the
// keys of one lane's operand each).  Eight lanes that read or write together (one chunk
// of 8 keys, 8 pieces of 16 columns of a key, one chunk of 8 columns) hit distinct banks.
__device__ __forceinline__ int k_slot(int key, int chunk) { return chunk ^ (key & 7) ^ (chunk >> 3 & 1); }
__device__ __forceinline__ int v_slot(int col, int chunk) { return chunk ^ (((col >> 2) ^ col) & 7); }

template <int CODE, int J, int RB, int W>
__global__ __launch_bounds__(64 * W, W / 4) void kv8_attn_tile(const ktir_kv8_attn_t d, uint32_t slots, int* err) {
  constexpr int TM = 32 * RB * W, DP = 64 * J, NT = 64 * W;
  constexpr int KU = TILE_KEYS * 4 * J, VU = 16 * 16 * J, KP = (KU + NT - 1) / NT, VP = (VU + NT - 1) / NT;   // units of a step, a thread's
  constexpr bool TURNS = J == 2;                 // the two wavefronts of a SIMD take turns
  static_assert(J == 1 || J == 2 || J == 4, "columns in 64s");
  static_assert(!TURNS || W == 8, "two wavefronts of a SIMD: i and i + 4");
  __shared__ __attribute__((aligned(16))) uint16_t ks[2][TILE_KEYS * DP], vs[2][DP * TILE_KEYS];
  const ktir_kv8_t& c = d.cache;
  const int tid = threadIdx.x, l = tid & 63, wave = uni(tid >> 6), h = l >> 5, r32 = l & 31;
  const int grp = (int)((uint32_t)d.q_heads / (uint32_t)c.heads), D = (int)c.columns, shift = __builtin_ctz((uint32_t)c.page);
  // a head's tiles share one XCD's L2 where there are 8 heads; the longest rows (the last tiles) start first
  const uint32_t heads = (uint32_t)c.heads, order = blockIdx.x / heads, slot = slots - 1 - order;
  const int64_t head = blockIdx.x - order * heads;
  const Tile t = uni(tile_of(d, slot, TM, grp, err));
  if (!t.rows) return;
  const int from = t.lo & ~(TILE_KEYS - 1);

  // this lane's rows; the wavefront's bounds of keys
  const int w0 = t.row0 + wave * 32 * RB, wn = t.rows - wave * 32 * RB < 32 * RB ? t.rows - wave * 32 * RB : 32 * RB;
  int see_lo[RB], lo_most = 0, hi_least = 0, other;
  uint32_t see[RB];                                  // how many keys a row sees, from see_lo on
  uint4 qf[RB][4 * J];
  float rs[RB];
  const bool whole = !((d.q.ptr | (uint64_t)d.q.tok * 2 | (uint64_t)d.q.head * 2) & 15);
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    int r = w0 + 32 * b + r32;
    if (r >= t.row0 + t.rows) r = t.row0 + t.rows - 1;            // a row that is not stored
    int see_hi;
    seen(d, t, r, grp, &see_lo[b], &see_hi);
    see[b] = see_hi > see_lo[b] ? see_hi - see_lo[b] : 0;
    const int64_t e = (t.q.start + r / grp) * d.q.tok + (head * grp + r % grp) * d.q.head;
    uint32_t raw[4 * J][4], top = 0;
#pragma unroll
    for (int s = 0; s < 4 * J; ++s) {
      const int x = 16 * s + 8 * h;
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[s][i] = 0;
      if (x < D) {
        const KTIR_G(uint16_t)* p = (const KTIR_G(uint16_t)*)d.q.ptr + e + x;
        if (whole) {
          const u32x4_t a = *(const KTIR_G(u32x4_t)*)p;
#pragma unroll
          for (int i = 0; i < 4; ++i) raw[s][i] = a[i];
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) raw[s][i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
        }
      }
    }
#pragma unroll
    for (int s = 0; s < 4 * J; ++s) top = top_bits(raw[s], top);
    const uint32_t half = __shfl_xor(top, 32);
    top = top > half ? top : half;
    const int up = d.dtype == KTIR_BF16 ? q_power(top) : 0;
    rs[b] = power2(-up) * (d.scale * LOG2E);
#pragma unroll
    for (int s = 0; s < 4 * J; ++s) {
      if (d.dtype == KTIR_BF16) q_scaled(raw[s], power2(up));
      qf[b][s] = make_uint4(raw[s][0], raw[s][1], raw[s][2], raw[s][3]);
    }
  }
  if (wn > 0) {
    seen(d, t, w0, grp, &other, &hi_least);
    seen(d, t, w0 + wn - 1, grp, &lo_most, &other);
  }
  lo_most = uni(lo_most), hi_least = uni(hi_least);

  f32x16_t acc[RB][2 * J];
  float base[RB], sum[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    base[b] = B_NONE;
    sum[b] = 0.f;
#pragma unroll
    for (int n = 0; n < 2 * J; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[b][n][i] = 0.f;
  }

  // a thread's share of a step: units of 16 codes of a key, and of 4 columns of 4 keys of V
  const uint32_t seen_by_some = t.hi > t.lo ? t.hi - t.lo : 0;      // keys, from t.lo on
  const int steps = t.hi > from ? (t.hi - from + TILE_KEYS - 1) / TILE_KEYS : 0;
  // the groups of the 16 steps that the computed one is of, of those that keys are fetched of (four steps on), and the next
  KV8Groups cur = {0, 0.f, 0.f, L_UNIT}, g = cur, next = cur;
  u32x4_t k_raw[2][KP];                               // of even and odd steps
  uint32_t v_raw[2][VP][4];
  auto page_of = [&](int pages, int j, int group) { return (int64_t)__builtin_amdgcn_readlane(pages, 4 * (j & 15) + (group & 3)); };
  // key of a K unit, first key of a V unit: one group of 16 a wavefront
  auto k_key = [&](int p) { return (tid + NT * p) / (4 * J); };
  // (a V unit is half a chunk of 4 columns: 8 column fours, both halves, the other fours, the chunks)
  auto v_chunk = [&](int p) { return (tid + NT * p) / (32 * J); };
  const int v_half = tid >> 3 & 1;
  auto v_col = [&](int p) { return ((tid & 7) + 8 * ((tid + NT * p) / 16 % (2 * J))) * 4; };
  auto v_key = [&](int p) { return 16 * (v_chunk(p) >> 1) + 4 * (v_chunk(p) & 1) + 8 * v_half; };
  auto fetch_k = [&](int j, u32x4_t (&kraw)[KP]) {
    const int key = from + TILE_KEYS * j;
#pragma unroll
    for (int p = 0; p < KP; ++p) {
      // (columns behind D: the first ones again, times zeros in Q)
      const int r = k_key(p), at = (tid + NT * p) % (4 * J) * 16, col = at < D ? at : 0;
      const uint64_t page = c.k + page_of(g.page, j, uni(r >> 4)) * c.k_page + head * c.k_head;
      const uint32_t at32 = (uint32_t)((key + r) & (int)(c.page - 1)) * (uint32_t)c.k_tok + col;    // (tokens of a page lie 2^22 bytes apart at most)
      if (KU % NT == 0 || tid < KU) kraw[p] = *(const KTIR_G(u32x4_t)*)((const KTIR_G(char)*)page + at32);
    }
  };
  auto fetch_v = [&](int j, int pages, uint32_t (&vraw)[VP][4]) {
    const int key = from + TILE_KEYS * j;
#pragma unroll
    for (int p = 0; p < VP; ++p) {
      // (columns behind D: the first ones again, not stored)
      const int first = v_key(p), x = v_col(p), col = x < D ? x : 0;
      const uint64_t page = c.v + page_of(pages, j, uni(first >> 4)) * c.v_page + head * c.v_head;
      const uint32_t at32 = (uint32_t)((key + first) & (int)(c.page - 1)) * (uint32_t)c.v_tok + col;
      if (VU % NT == 0 || tid < VU) {
#pragma unroll
        for (int i = 0; i < 4; ++i) vraw[p][i] = *(const KTIR_G(uint32_t)*)((const KTIR_G(char)*)(page + i * c.v_tok) + at32);
      }
    }
  };
  auto put_k = [&](int buf, const u32x4_t (&kraw)[KP]) {
    uint16_t* kb = ks[buf];
#pragma unroll
    for (int p = 0; p < KP; ++p) {
      if (KU % NT && tid >= KU) break;
      const int r = k_key(p), chunk = (tid + NT * p) % (4 * J) * 2;
      *(uint4*)(kb + r * DP + 8 * k_slot(r, chunk)) = row_half8<CODE>(kraw[p].x, kraw[p].y);
      *(uint4*)(kb + r * DP + 8 * k_slot(r, chunk + 1)) = row_half8<CODE>(kraw[p].z, kraw[p].w);
    }
  };
  auto put_v = [&](int j, int buf, uint32_t (&vraw)[VP][4]) {
    uint16_t* vb = vs[buf];
#pragma unroll
    for (int p = 0; p < VP; ++p) {
      if (VU % NT && tid >= VU) break;
      const int chunk = v_chunk(p), col = v_col(p);
      if (CODE == KTIR_E4M3) {                    // NaN codes of tokens that no row sees
        const int first = from + TILE_KEYS * j + v_key(p) - t.lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) vraw[p][i] = (uint32_t)(first + i) < seen_by_some ? vraw[p][i] : 0u;
      }
      uint32_t a[4], b[4];
      cross_half2<CODE>(vraw[p][0], vraw[p][1], a);
      cross_half2<CODE>(vraw[p][2], vraw[p][3], b);
#pragma unroll
      for (int n = 0; n < 4; ++n)
        *(uint2*)(vb + (col + n) * TILE_KEYS + 8 * v_slot(col + n, chunk) + 4 * v_half) = make_uint2(a[n], b[n]);
    }
  };
  const f32x16_t zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  // scores of a step, K rows times Q, of columns 16 first .. 16 (first + n)
  auto scores = [&](f32x16_t (&s)[RB][2], int buf, int first, int n) {
    const uint16_t* kb = ks[buf];
#pragma unroll
    for (int x = first; x < first + n; ++x)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint4 a = *(const uint4*)(kb + (32 * k + r32) * DP + 8 * k_slot(32 * k + r32, 2 * x + h));
#pragma unroll
        for (int b = 0; b < RB; ++b) s[b][k] = mfma_at<false>(a, qf[b][x], x ? s[b][k] : zero);
      }
  };
  auto top_of = [&](const f32x16_t (&x)[2]) {
    float top = x[0][0];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, x[k][i]);
    return top;
  };
  f32x16_t s0[RB][2], s1[RB][2];                 // scores of even and odd steps
  if (steps) {
    const bool there = kv8_there(t, from + 16 * l);
    g = kv8_groups(d, head, kv8_pages(d, t, from + 16 * l, shift), there, err);
    kv8_scales(g, there);
    cur = g;
    fetch_k(0, k_raw[0]);
    fetch_v(0, g.page, v_raw[0]);
    fetch_k(1, k_raw[1]);              // (steps past the last: page 0)
    fetch_v(1, g.page, v_raw[1]);
    put_k(0, k_raw[0]);
    put_v(0, 0, v_raw[0]);
    put_k(1, k_raw[1]);
    fetch_k(2, k_raw[0]);
    fetch_v(2, g.page, v_raw[0]);
    fetch_k(3, k_raw[1]);
    __syncthreads();
    scores(s0, 0, 0, 4 * J);
    __syncthreads();
  }

  // Step j: its scores are in s, those of step j + 1 go to s_next; PAR is j's parity, so that the
  // buffers' addresses do not change.
  auto step = [&](int j, auto parity, f32x16_t (&s)[RB][2], f32x16_t (&s_next)[RB][2]) {
    constexpr int PAR = decltype(parity)::value;
    // the next 16 steps' groups: their pages four steps ahead of the first fetch, then the scales
    const int f = j + 4, key = from + TILE_KEYS * j;
    if ((f & 15) == 12) next.page = kv8_pages(d, t, from + TILE_KEYS * (f + 4) + 16 * l, shift);
    if ((f & 15) == 14) next = kv8_groups(d, head, next.page, kv8_there(t, from + TILE_KEYS * (f + 2) + 16 * l), err);
    const int vpages = (f & 15) == 0 ? cur.page : g.page;          // of step j + 3, in the 16 before g's next ones then
    if ((f & 15) == 0) {
      g = next;
      kv8_scales(g, kv8_there(t, from + TILE_KEYS * f + 16 * l));
    }
    if ((j & 15) == 0) cur = g;
    float gks[4], glv[4], giv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = 4 * (j & 15) + i;
      gks[i] = lane_of(cur.ks, at);
      glv[i] = lane_of(cur.lv, at);
      giv[i] = lane_of(cur.iv, at);
    }
    // exponents of the weights, less b
    const bool cut = key < lo_most || key + TILE_KEYS > hi_least;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      // (made anew in each of the two rare parts: kept, the 32 places take as many registers)
      auto places = [&]() {
        int first = key + 4 * h - see_lo[b];
        asm volatile("" : "+v"(first));
        return first;
      };
      auto hidden = [&](int first, int k, int i) { return (uint32_t)(first + 32 * k + 8 * (i >> 2) + (i & 3)) >= see[b]; };
      if (__any(base[b] == B_NONE)) {              // rows that have seen no key: b from this step's, their sums are 0
        float top = -__builtin_inff();
        const int first = places();
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            top = __builtin_fmaxf(top, mask_ninf(__builtin_fmaf(s[b][k][i], gks[2 * k + (i >> 3)] * rs[b], glv[2 * k + (i >> 3)]), hidden(first, k, i)));
        top = __builtin_fmaxf(top, other_half(top));
        base[b] = base[b] == B_NONE && top > -__builtin_inff() ? top - TILE_TOP : base[b];
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][k][i] = __builtin_fmaf(s[b][k][i], gks[2 * k + (i >> 3)] * rs[b], glv[2 * k + (i >> 3)] - base[b]);
      if (cut) {
        const int first = places();
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[b][k][i] = mask_ninf(s[b][k][i], hidden(first, k, i));
      }
    }
    float top[RB], most = -__builtin_inff();
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      top[b] = top_of(s[b]);
      most = __builtin_fmaxf(most, top[b]);
    }
    if (__any(most > TILE_TOP + TILE_LAG)) {
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        top[b] = __builtin_fmaxf(top[b], other_half(top[b]));
        const float by = top[b] > TILE_TOP ? top[b] - TILE_TOP : 0.f, keep = __builtin_amdgcn_exp2f(-by);
        base[b] += by;
        sum[b] *= keep;
#pragma unroll
        for (int n = 0; n < 2 * J; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[b][n][i] *= keep;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[b][k][i] -= by;
      }
    }
    // the codes of steps j + 2 (K) and j + 1 (V) into LDS, those of the next two steps on their way, the scores of j + 1,
    // beside W V of step j.  (Past the last step: of page 0, unused.)
    const uint16_t* vb = vs[PAR];
    auto move = [&](int p) {
      if (p == 0) put_k(PAR, k_raw[PAR]);
      if (p == 1) put_v(j + 1, 1 - PAR, v_raw[1 - PAR]);
      if (p == 2) fetch_k(j + 4, k_raw[PAR]);
      if (p == 3) fetch_v(j + 3, vpages, v_raw[1 - PAR]);
    };
    // w: the weights rounded, and what that leaves of them
    auto weights = [&](int p, uint4 (&w)[RB][2]) {
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        uint32_t t[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float e[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            e[k] = __builtin_amdgcn_exp2f(s[b][p >> 1][8 * (p & 1) + 2 * i + k]);
            sum[b] = __builtin_fmaf(e[k], giv[p], sum[b]);
          }
          t[0][i] = cvt2<false>(e[0], e[1]);
          const f16x2_t top = __builtin_bit_cast(f16x2_t, t[0][i]);
          t[1][i] = cvt2<false>(__builtin_fmaf((float)top.x, -1.f, e[0]), __builtin_fmaf((float)top.y, -1.f, e[1]));      // (one mixed fma each)
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) w[b][k] = make_uint4(t[k][0], t[k][1], t[k][2], t[k][3]);
      }
    };
    auto weigh = [&](int p, const uint4 (&w)[RB][2]) {
#pragma unroll
      for (int n = 0; n < 2 * J; ++n) {
        const uint4 a = *(const uint4*)(vb + (32 * n + r32) * TILE_KEYS + 8 * v_slot(32 * n + r32, 2 * p + h));
#pragma unroll
        for (int x = 1; x >= 0; --x)
#pragma unroll
          for (int b = 0; b < RB; ++b) acc[b][n] = mfma_at<false>(a, w[b][x], acc[b][n]);
      }
    };
    if constexpr (TURNS) {
      uint4 w[4][RB][2];
#pragma unroll
      for (int p = 0; p < 4; ++p) weights(p, w[p]);
      __builtin_amdgcn_sched_barrier(0);
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        move(p);
        scores(s_next, 1 - PAR, p * J, J);
        weigh(p, w[p]);
      }
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
    } else {
      uint4 w[RB][2], old[RB][2];
#pragma unroll
      for (int p = 0; p < 5; ++p) {
        if (J == 4 || p == 0 || p == 2 || p == 4) __builtin_amdgcn_sched_barrier(0);
        move(p);
        if (p < 4) scores(s_next, 1 - PAR, p * J, J);
#pragma unroll
        for (int b = 0; b < RB; ++b) old[b][0] = w[b][0], old[b][1] = w[b][1];
        if (p < 4) weights(p, w);
        if (p > 0) weigh(p - 1, old);
      }
    }
    __syncthreads();
  };
  // In turns the later half of the wavefronts, one of each SIMD, is a barrier behind the others, which reach as many in the
  // end.  A buffer is last read in a half that precedes the first in which any wavefront writes it again, and is whole a
  // half before it is read.
  if (TURNS && wave >= W / 2) __syncthreads();
  for (int j = 0; j < steps; j += 2) {
    step(j, std::integral_constant<int, 0>(), s0, TURNS ? s0 : s1);
    if (j + 1 < steps) step(j + 1, std::integral_constant<int, 1>(), TURNS ? s0 : s1, s0);
  }
  if (TURNS && wave < W / 2) __syncthreads();

  // O^T: a lane has columns 32 n + 8 g + 4 h + 0..3 of its row
  const bool packed = !((d.out.ptr | (uint64_t)d.out.tok * 2 | (uint64_t)d.out.head * 2) & 7);
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    const int r = w0 + 32 * b + r32;
    sum[b] += other_half(sum[b]);
    if (r >= t.row0 + t.rows) continue;
    const bool none = !see[b];
    const float inv = none ? 0.f : L_UNIT / sum[b];
    const int64_t tok = t.q.start + r / grp, hq = head * grp + r % grp, e = tok * d.out.tok + hq * d.out.head;
#pragma unroll
    for (int n = 0; n < 2 * J; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int x = 32 * n + 8 * q + 4 * h;
        if (x >= D) continue;
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = none ? 0.f : acc[b][n][4 * q + i] * inv;
        if (packed) {
          const u32x2_t v = d.dtype == KTIR_BF16 ? u32x2_t{cvt2<true>(o[0], o[1]), cvt2<true>(o[2], o[3])}
                                                 : u32x2_t{cvt2<false>(o[0], o[1]), cvt2<false>(o[2], o[3])};
          *(KTIR_G(u32x2_t)*)((KTIR_G(uint16_t)*)d.out.ptr + e + x) = v;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) store_elem(d.out.ptr, e + x + i, d.dtype, o[i]);
        }
      }
    if (d.lse && h == 0)
      ((KTIR_G(float)*)d.lse)[tok * d.lse_tok + hq * d.lse_head] =
          none ? -__builtin_inff() : (base[b] + 16.f + __builtin_amdgcn_logf(sum[b])) * 0.69314718055994530942f;
  }
}

template <int CODE>
static void tile_go(const ktir_kv8_attn_t& d, int64_t slots, hipStream_t st) {
  const dim3 grid((unsigned)(slots * d.cache.heads));
  const int D = (int)d.cache.columns;
  if (D <= 64) hipLaunchKernelGGL((kv8_attn_tile<CODE, 1, 1, 8>), grid, dim3(512), 0, st, d, (uint32_t)slots, device_error_flag());
  else if (D <= 128) hipLaunchKernelGGL((kv8_attn_tile<CODE, 2, 1, 8>), grid, dim3(512), 0, st, d, (uint32_t)slots, device_error_flag());
  else hipLaunchKernelGGL((kv8_attn_tile<CODE, 4, 1, 4>), grid, dim3(256), 0, st, d, (uint32_t)slots, device_error_flag());
}

// Whether a launch takes this kernel, and its tiles of rows for each KV head.  With fewer
// than 128 workgroups the kernel of few rows, which spreads the keys as well, is faster (128
// columns): the last 512 of 4096 tokens (72 tiles) 86 us there and 156 here, the last 700 (88) 120
// and 157, the last 1024 (136) 148 and 157, the last 1400 (176) 202 and 164, 2048 alone (264) 120 and 93,
// 16 sequences of 64 after 1984 (128) 103 and 92, 20 (160) 125 and 90.  With 64 columns 16 sequences (128)
// take 75 and 73, the last 1024 (136) 114 and 123; with 256 this kernel gains later: the last 512 (136)
// 176 and 273, 8 sequences of 300 after 1700 (332) 249 and 275, 32 of 40 after 960 (576) 216 and 171.  And the
// kernel of few rows is where no tile is more than half full: 16 sequences of 20 (80 rows of 256) 50 and 87.
bool kv8_tile_takes(const ktir_kv8_attn_t& d, int64_t* slots) {
  const int64_t grp = d.q_heads / d.cache.heads, TM = d.cache.columns <= 128 ? 256 : 128;
  if (d.max_q * grp <= TM / 2) return false;
  *slots = d.max_q * grp > TM ? d.batch.tokens * grp / TM + d.batch.seqs : d.batch.seqs;
  return *slots * d.cache.heads >= 128;
}

int kv8_tile_launch(const ktir_kv8_attn_t& d, int64_t slots) {
  d.cache.dtype == KTIR_I8 ? tile_go<KTIR_I8>(d, slots, stream_of(d.stream)) : tile_go<KTIR_E4M3>(d, slots, stream_of(d.stream));
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}

}  // namespace ktir
