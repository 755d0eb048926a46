// Attention over the 8-bit cache for many rows: prompts and chunks of them.
//
// A workgroup has 128 RB rows (tokens x the query heads of one KV head) of one
// sequence, 32 RB of them in each of its four wavefronts, and runs over the keys that
// they see, 64 at a time.  The codes of a step are made f16 once for all rows and
// laid into LDS (two buffers): K as [key][column], V as [column][key], with the keys
// of each 16 in the order that the scores' layout leaves them in:
//   S^T = K Q^T     32 x 32 x 16 MFMA, one row a lane (the two halves share it)
//   w, b, l         as ktir_kv8_dev.h says; w enters the product as one f16 term
//   O^T += V^T W^T  no exchange between lanes
// With RB = 2 a fragment read from LDS serves two products; one wavefront a SIMD
// then has its 512 registers.
//
// One f16 term: w is at most 2^15 and normal down to 2^-14, so a key keeps 11 bits
// (the result's own, in f16) unless the row's heaviest one outweighs it 2^25 to 2^29
// times; less is added with the step of 2^-24, which is 2^-35 to 2^-39 of the heaviest.
#include "ktir_kv8_dev.h"

namespace ktir {

constexpr int TILE_KEYS = 64, TILE_WAVES = 4, TILE_GROUPS = 64;
constexpr float TILE_TOP = 11.f, TILE_LAG = 4.f;       // exponent of the largest weight when b changes, and by how much it may grow

template <int CODE, int J, int RB>
struct TileRaw {
  u32x4_t k[J];          // J pieces of 16 codes of a key
  uint32_t v[J > 2 ? J / 2 : 1][8];      // 4 columns of 8 keys, (J + 1) / 2 times
};

// chunk slots in LDS: 16 bytes, 8 of a K row's (of 8 J), 8 of a V column's 64 keys
__device__ __forceinline__ int k_slot(int key, int chunk) { return chunk ^ (key & 7); }
__device__ __forceinline__ int v_slot(int col, int chunk) { return chunk ^ (((col >> 2) ^ col) & 7); }

template <int CODE, int J, int RB>
__global__ __launch_bounds__(256, 1) void kv8_attn_tile(const ktir_kv8_attn_t d, uint32_t slots, int* err) {
  constexpr int TM = 128 * RB, DP = 64 * J, VU = J > 2 ? J / 2 : 1;
  static_assert(J == 1 || J == 2 || J == 4, "columns in 64s");
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
  int see_lo[RB], see_hi[RB], lo_least = 0, lo_most = 0, hi_least = 0, hi_most = 0;
  uint4 qf[RB][4 * J];
  float rs[RB];
  const bool whole = !((d.q.ptr | (uint64_t)d.q.tok * 2 | (uint64_t)d.q.head * 2) & 15);
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    int r = w0 + 32 * b + r32;
    if (r >= t.row0 + t.rows) r = t.row0 + t.rows - 1;            // a row that is not stored
    seen(d, t, r, grp, &see_lo[b], &see_hi[b]);
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
    const uint32_t other = __shfl_xor(top, 32);
    top = top > other ? top : other;
    const int up = d.dtype == KTIR_BF16 ? q_power(top) : 0;
    rs[b] = power2(-up) * (d.scale * LOG2E);
#pragma unroll
    for (int s = 0; s < 4 * J; ++s) {
      if (d.dtype == KTIR_BF16) q_scaled(raw[s], power2(up));
      qf[b][s] = make_uint4(raw[s][0], raw[s][1], raw[s][2], raw[s][3]);
    }
  }
  if (wn > 0) {
    seen(d, t, w0, grp, &lo_least, &hi_least);
    seen(d, t, w0 + wn - 1, grp, &lo_most, &hi_most);
  }
  lo_least = uni(lo_least), lo_most = uni(lo_most), hi_least = uni(hi_least), hi_most = uni(hi_most);

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

  // this thread's share of a step: J pieces of 16 codes of keys (tid / (4 J) + 64 / J p), and 4 columns of the 8 keys of one V chunk
  KV8Groups g = {0, 0.f, 0.f, L_UNIT};
  TileRaw<CODE, J, RB> raw;
  const int kkey = tid / (4 * J), kcol = tid % (4 * J) * 16;
  auto fetch = [&](int key) {                     // the groups of the step at `key` are in lanes ((key - from) / 16) % 64 of g
    const int group = ((key - from) >> 4) & (TILE_GROUPS - 1);
#pragma unroll
    for (int p = 0; p < J; ++p) {
      const int r = kkey + 64 / J * p;
      // keys of a wavefront's piece lie in one group of 16: 64 / (4 J) of them, from a multiple of that on
      const int64_t page = __builtin_amdgcn_readlane(g.page, group + uni(r >> 4)), row = (key + r) & (c.page - 1);
      if (kcol < D) raw.k[p] = *(const KTIR_G(u32x4_t)*)(c.k + page * c.k_page + row * c.k_tok + head * c.k_head + kcol);
    }
#pragma unroll
    for (int p = 0; p < VU; ++p) {
      const int unit = tid + 256 * p, chunk = unit / (16 * J), col = unit % (16 * J) * 4;
      const int first = (16 * (chunk >> 1) + 4 * (chunk & 1)) & (TILE_KEYS - 1);
      // (a wavefront has one group, two with 64 columns)
      const int64_t page = J == 1 ? __shfl(g.page, group + (first >> 4)) : __builtin_amdgcn_readlane(g.page, group + uni(first >> 4));
      if (unit < 8 * 16 * J) {
        const uint64_t at = c.v + page * c.v_page + head * c.v_head + col;
        const int64_t row = (key + first) & (c.page - 1);
        if (col < D) {
#pragma unroll
          for (int i = 0; i < 8; ++i) raw.v[p][i] = *(const KTIR_G(uint32_t)*)(at + (row + (i & 3) + 8 * (i >> 2)) * c.v_tok);
        }
      }
    }
  };
  auto put = [&](int key, uint16_t* kb, uint16_t* vb) {
#pragma unroll
    for (int p = 0; p < J; ++p) {
      const int r = kkey + 64 / J * p, chunk = kcol / 8;
      *(uint4*)(kb + r * DP + 8 * k_slot(r, chunk)) = row_half8<CODE>(raw.k[p].x, raw.k[p].y);
      *(uint4*)(kb + r * DP + 8 * k_slot(r, chunk + 1)) = row_half8<CODE>(raw.k[p].z, raw.k[p].w);
    }
#pragma unroll
    for (int p = 0; p < VU; ++p) {
      const int unit = tid + 256 * p, chunk = unit / (16 * J), col = unit % (16 * J) * 4;
      if (unit >= 8 * 16 * J) break;
      if (CODE == KTIR_E4M3 && key + TILE_KEYS > t.hi) {            // NaN codes of tokens that no row sees
        const int first = key + 16 * (chunk >> 1) + 4 * (chunk & 1);
#pragma unroll
        for (int i = 0; i < 8; ++i) raw.v[p][i] = first + (i & 3) + 8 * (i >> 2) < t.hi ? raw.v[p][i] : 0u;
      }
      uint32_t o[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) cross_half2<CODE>(raw.v[p][2 * i], raw.v[p][2 * i + 1], o[i]);
#pragma unroll
      for (int n = 0; n < 4; ++n)
        *(uint4*)(vb + (col + n) * TILE_KEYS + 8 * v_slot(col + n, chunk)) = make_uint4(o[0][n], o[1][n], o[2][n], o[3][n]);
    }
  };
  int g_from = from;
  auto groups = [&](int key) {                    // of the 64 groups from `key` on
    g_from = key;
    const bool there = key + 16 * l < t.hi;
    g = kv8_groups(d, head, kv8_pages(d, t, key + 16 * l, t.hi, shift), there, err);
    kv8_scales(g, there);
  };

#pragma unroll
  for (int p = 0; p < J; ++p) raw.k[p] = u32x4_t{0, 0, 0, 0};         // columns behind D
#pragma unroll
  for (int p = 0; p < VU; ++p)
#pragma unroll
    for (int i = 0; i < 8; ++i) raw.v[p][i] = 0;
  KV8Groups now = g;                              // the groups of the step that is computed
  if (from < t.hi) {
    groups(from);
    now = g;
    fetch(from);
    put(from, ks[0], vs[0]);
    if (from + TILE_KEYS < t.hi) fetch(from + TILE_KEYS);
  }
  __syncthreads();

  int buf = 0;
  for (int key = from; key < t.hi; key += TILE_KEYS, buf ^= 1) {
    const int group = ((key - from) >> 4) & (TILE_GROUPS - 1);
    if (key + TILE_KEYS < t.hi) {
      put(key + TILE_KEYS, ks[buf ^ 1], vs[buf ^ 1]);
      if (key + 2 * TILE_KEYS < t.hi) {
        if (!(((key + 2 * TILE_KEYS - from) >> 4) & (TILE_GROUPS - 1))) {
          now = g;
          groups(key + 2 * TILE_KEYS);
        }
        fetch(key + 2 * TILE_KEYS);
      }
    }
    if (key < hi_most && key + TILE_KEYS > lo_least && wn > 0) {
      const uint16_t *kb = ks[buf], *vb = vs[buf];
      f32x16_t s[RB][2];
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[b][k][i] = 0.f;
#pragma unroll
      for (int x = 0; x < 4 * J; ++x)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint4 a = *(const uint4*)(kb + (32 * k + r32) * DP + 8 * k_slot(32 * k + r32, 2 * x + h));
#pragma unroll
          for (int b = 0; b < RB; ++b) s[b][k] = mfma_at<false>(a, qf[b][x], s[b][k]);
        }
      const bool old = key < g_from;
      float gks[4], glv[4], giv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        gks[i] = lane_of(old ? now.ks : g.ks, group + i);
        glv[i] = lane_of(old ? now.lv : g.lv, group + i);
        giv[i] = lane_of(old ? now.iv : g.iv, group + i);
      }
      uint4 w[RB][4];
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        // exponents of the weights, less b
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int gi = 2 * k + (i >> 3);
            s[b][k][i] = __builtin_fmaf(s[b][k][i], gks[gi] * rs[b], glv[gi]);
          }
        const bool cut = key < lo_most || key + TILE_KEYS > hi_least;
        if (cut) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int j = key + 32 * k + 8 * (i >> 2) + 4 * h + (i & 3);
              s[b][k][i] = mask_ninf(s[b][k][i], j < see_lo[b] || j >= see_hi[b]);
            }
        }
        float top = s[b][0][0];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, s[b][k][i]);
        if (__any(top > base[b] + (TILE_TOP + TILE_LAG))) {
          top = __builtin_fmaxf(top, other_half(top));
          const float to = __builtin_fmaxf(base[b], top - TILE_TOP), keep = __builtin_amdgcn_exp2f(base[b] - to);
          base[b] = to;
          sum[b] *= keep;
#pragma unroll
          for (int n = 0; n < 2 * J; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[b][n][i] *= keep;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float e = __builtin_amdgcn_exp2f(s[b][k][i] - base[b]);
            sum[b] = __builtin_fmaf(e, giv[2 * k + (i >> 3)], sum[b]);
            s[b][k][i] = e;
          }
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const f32x16_t& x = s[b][p >> 1];
          const int i = 8 * (p & 1);
          w[b][p] = make_uint4(cvt2<false>(x[i], x[i + 1]), cvt2<false>(x[i + 2], x[i + 3]), cvt2<false>(x[i + 4], x[i + 5]),
                               cvt2<false>(x[i + 6], x[i + 7]));
        }
      }
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int n = 0; n < 2 * J; ++n) {
          const uint4 a = *(const uint4*)(vb + (32 * n + r32) * TILE_KEYS + 8 * v_slot(32 * n + r32, 2 * p + h));
#pragma unroll
          for (int b = 0; b < RB; ++b) acc[b][n] = mfma_at<false>(a, w[b][p], acc[b][n]);
        }
    }
    __syncthreads();
  }

  // O^T: a lane has columns 32 n + 8 g + 4 h + 0..3 of its row
  const bool packed = !((d.out.ptr | (uint64_t)d.out.tok * 2 | (uint64_t)d.out.head * 2) & 7);
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    const int r = w0 + 32 * b + r32;
    sum[b] += other_half(sum[b]);
    if (r >= t.row0 + t.rows) continue;
    const bool none = see_lo[b] >= see_hi[b];
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
  if (D <= 64) hipLaunchKernelGGL((kv8_attn_tile<CODE, 1, 2>), grid, dim3(256), 0, st, d, (uint32_t)slots, device_error_flag());
  else if (D <= 128) hipLaunchKernelGGL((kv8_attn_tile<CODE, 2, 2>), grid, dim3(256), 0, st, d, (uint32_t)slots, device_error_flag());
  else hipLaunchKernelGGL((kv8_attn_tile<CODE, 4, 1>), grid, dim3(256), 0, st, d, (uint32_t)slots, device_error_flag());
}

// whether a launch takes this kernel, and its tiles of rows for each KV head
bool kv8_tile_takes(const ktir_kv8_attn_t& d, int64_t* slots) {
  const int64_t grp = d.q_heads / d.cache.heads, TM = d.cache.columns <= 128 ? 256 : 128;
  if (d.max_q * grp <= TM / 2) return false;
  *slots = d.max_q * grp > TM ? d.batch.tokens * grp / TM + d.batch.seqs : d.batch.seqs;
  return *slots * d.cache.heads >= 160;
}

int kv8_tile_launch(const ktir_kv8_attn_t& d, int64_t slots) {
  d.cache.dtype == KTIR_I8 ? tile_go<KTIR_I8>(d, slots, stream_of(d.stream)) : tile_go<KTIR_E4M3>(d, slots, stream_of(d.stream));
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}

}  // namespace ktir
