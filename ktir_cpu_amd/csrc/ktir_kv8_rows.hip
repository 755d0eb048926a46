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
// lane, so no step waits for the chain table -> page -> key; the codes of the next
// step are in flight while this one is computed.
#include "ktir_kv8_dev.h"

namespace ktir {

constexpr int ROWS_WAVES = 4, ROWS_STEP = 32, ROWS_GROUPS = 64;

// what a split of a tile leaves in the workspace: TM rows of 64 J sums, then b and l of each row
template <int J, int MT>
constexpr int64_t PART = 16 * MT * (64 * J + 2);

template <int J>
struct KV8Step {
  u32x4_t k[2][J];
  uint32_t v[8][J];
};

// where a wavefront's next 64 groups of 16 keys lie, a group per lane
struct KV8Groups {
  int page;             // of the cache
  float ks, lv, iv;     // kscale, log2 vscale, 2^-16 / vscale
};

__device__ __forceinline__ float lane_of(float x, int i) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), i));
}

__device__ __forceinline__ KV8Groups kv8_groups(const ktir_kv8_attn_t& d, const Tile& t, int64_t head, int key, int end, int shift,
                                                int* err) {
  KV8Groups g = {0, 0.f, 0.f, 1.f};
  if (key < end) {
    const int64_t at = ints(d.batch.table)[t.s * d.batch.table_row + (key >> shift)];
    if (at < 0 || at >= d.cache.pages) *err = OUT_OF_RANGE;
    else g.page = (int)at;
    g.ks = ((const KTIR_G(float)*)d.cache.k_scale)[g.page * d.cache.ks_page + head * d.cache.ks_head];
    float vs = ((const KTIR_G(float)*)d.cache.v_scale)[g.page * d.cache.vs_page + head * d.cache.vs_head];
    vs = vs < LEAST_V ? LEAST_V : vs;
    g.lv = __builtin_amdgcn_logf(vs);
    g.iv = L_UNIT / vs;
  }
  return g;
}

// the codes of 32 keys from `key` on; groups that the wavefront does not have read page 0
template <int J>
__device__ __forceinline__ void kv8_load(const ktir_kv8_t& c, const KV8Groups& g, int group, int key, int64_t head, int koff, int voff,
                                         const int (&kpiece)[J], KV8Step<J>& o) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t page = __builtin_amdgcn_readlane(g.page, group + h);
    const int64_t row = (key + 16 * h) & (c.page - 1);
    const KTIR_G(uint8_t)* kp = (const KTIR_G(uint8_t)*)c.k + page * c.k_page + row * c.k_tok + head * c.k_head;
    const KTIR_G(uint8_t)* vp = (const KTIR_G(uint8_t)*)c.v + page * c.v_page + row * c.v_tok + head * c.v_head;
#pragma unroll
    for (int j = 0; j < J; ++j) o.k[h][j] = *(const KTIR_G(u32x4_t)*)(kp + (uint32_t)(koff + kpiece[j]));
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
__global__ __launch_bounds__(256) void kv8_attn_rows(const ktir_kv8_attn_t d, int* err) {
  constexpr int TM = 16 * MT, N = 4 * J, PITCH = 64 * J + 4;
  __shared__ __attribute__((aligned(16))) float o_sum[TM * PITCH];
  __shared__ float w_b[ROWS_WAVES][TM], w_l[ROWS_WAVES][TM];
  const ktir_kv8_t& c = d.cache;
  const int l = threadIdx.x & 63, wave = uni((int)(threadIdx.x >> 6)), g4 = l >> 4, c16 = l & 15;
  const int grp = (int)(d.q_heads / c.heads), D = (int)c.columns, shift = __builtin_ctz((uint32_t)c.page);
  const int splits = d.splits < 1 ? 1 : d.splits, split = (int)(blockIdx.x % splits);
  const int64_t item = blockIdx.x / splits, head = item % c.heads, slot = item / c.heads;
  const Tile t = tile_of(d, slot, TM, grp, err);
  if (!t.rows) return;

  // this workgroup's keys, and this wavefront's
  const int from = t.lo & ~(ROWS_STEP - 1), span = t.hi > from ? t.hi - from : 0;
  constexpr int QUANT = ROWS_STEP * ROWS_WAVES;
  const int part = ((span + splits - 1) / splits + QUANT - 1) / QUANT * QUANT, active = span ? (span + part - 1) / part : 1;
  if (split >= active) return;
  const int lo = uni(from + split * part + wave * (part / ROWS_WAVES)), end = uni(lo + part / ROWS_WAVES < t.hi ? lo + part / ROWS_WAVES : t.hi);

  // Q: this lane's row of each 16, pieces g4, g4 + 4, .. of 16 columns; times 2^k, so that the row's largest value has exponent 14
  uint4 qf[MT][J][2];
  float rs[MT];
  int see_lo[MT], see_hi[MT], kpiece[J];
#pragma unroll
  for (int j = 0; j < J; ++j) kpiece[j] = (4 * j + g4) * 16 < D ? (4 * j + g4) * 16 : 0;
  const bool whole = !((d.q.ptr | (uint64_t)d.q.tok * 2 | (uint64_t)d.q.head * 2) & 15);
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    int r = t.row0 + 16 * m + c16;
    if (r >= t.row0 + t.rows) r = t.row0 + t.rows - 1;              // a row that is not stored
    seen(d, t, r, grp, &see_lo[m], &see_hi[m]);
    const int64_t e = (t.q.start + r / grp) * d.q.tok + (head * grp + r % grp) * d.q.head;
    uint32_t raw[J][8];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int x = (4 * j + g4) * 16;
#pragma unroll
      for (int i = 0; i < 8; ++i) raw[j][i] = 0;
      if (x < D) {
        const KTIR_G(uint16_t)* p = (const KTIR_G(uint16_t)*)d.q.ptr + e + x;
        if (whole) {
          const u32x4_t a = ((const KTIR_G(u32x4_t)*)p)[0], b = ((const KTIR_G(u32x4_t)*)p)[1];
#pragma unroll
          for (int i = 0; i < 4; ++i) raw[j][i] = a[i], raw[j][4 + i] = b[i];
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) raw[j][i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t a = raw[j][i] & 0x7fffu, b = (raw[j][i] >> 16) & 0x7fffu;
        top = top > a ? top : a;
        top = top > b ? top : b;
      }
    }
    const bool bf = d.dtype == KTIR_BF16;
    {
      uint32_t y = __shfl_xor(top, 16);
      top = top > y ? top : y;
      y = __shfl_xor(top, 32);
      top = top > y ? top : y;
    }
    // f16 queries are operands as they are; bf16 ones take the power of two that brings the largest to 2^14
    int k = 0;
    if (bf && top) {
      k = 14 - ((int)(top >> 7) - 127);
      k = k > 120 ? 120 : k < -113 ? -113 : k;
    }
    const float up = __uint_as_float((uint32_t)(127 + k) << 23);
    rs[m] = __uint_as_float((uint32_t)(127 - k) << 23) * (d.scale * LOG2E);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (bf) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const f32x2_t v = uncvt2<true>(raw[j][i]);
          raw[j][i] = cvt2<false>(v.x * up, v.y * up);
        }
      }
      qf[m][j][0] = make_uint4(raw[j][0], raw[j][1], raw[j][2], raw[j][3]);
      qf[m][j][1] = make_uint4(raw[j][4], raw[j][5], raw[j][6], raw[j][7]);
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
  const int koff = c16 * (int)c.k_tok, vcol = c16 * 4 * J + 4 * J <= D ? c16 * 4 * J : 0, voff = 4 * g4 * (int)c.v_tok + vcol;

  auto step = [&](const KV8Step<J>& o, const KV8Groups& g, int group, int key) {
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
      float u[8], inv[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float f = ks[h] * rs[m];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[4 * h + i] = __builtin_fmaf(s[m][h][i], f, lv[h]), inv[4 * h + i] = iv[h];
      }
      if (cut) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int j = key + 16 * (i >> 2) + 4 * g4 + (i & 3);
          const bool out = j < see_lo[m] || j >= see_hi[m];
          u[i] = out ? -__builtin_inff() : u[i];
          inv[i] = out ? 0.f : inv[i];
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
        sum[m] = __builtin_fmaf(a, inv[i], sum[m]);
        sum[m] = __builtin_fmaf(e, inv[i + 1], sum[m]);
        hi[i / 2] = cvt2<true>(a, e);
        const f32x2_t back = uncvt2<true>(hi[i / 2]);
        lo_[i / 2] = cvt2<true>(a - back.x, e - back.y);
      }
      wh[m] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      wl[m] = make_uint4(lo_[0], lo_[1], lo_[2], lo_[3]);
    }
    uint32_t v[8][J];
    const bool tail = CODE == KTIR_E4M3 && key + ROWS_STEP > t.hi;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < J; ++j) v[i][j] = tail && key + 16 * (i >> 2) + 4 * g4 + (i & 3) >= t.hi ? 0u : o.v[i][j];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      uint32_t p[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) cross_bf2<CODE>(v[2 * i][j], v[2 * i + 1][j], p[i]);
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

  for (int base = lo; base < end; base += 16 * ROWS_GROUPS) {
    const KV8Groups g = kv8_groups(d, t, head, base + 16 * l, end, shift, err);
    const int n = (end - base + ROWS_STEP - 1) / ROWS_STEP, steps = n < ROWS_GROUPS / 2 ? n : ROWS_GROUPS / 2;
    KV8Step<J> o[2];
    kv8_load<J>(c, g, 0, base, head, koff, voff, kpiece, o[0]);
    for (int i = 0; i < steps; i += 2) {
      if (i + 1 < steps) kv8_load<J>(c, g, 2 * i + 2, base + ROWS_STEP * (i + 1), head, koff, voff, kpiece, o[1]);
      step(o[0], g, 2 * i, base + ROWS_STEP * i);
      if (i + 1 < steps) {
        if (i + 2 < steps) kv8_load<J>(c, g, 2 * i + 4, base + ROWS_STEP * (i + 2), head, koff, voff, kpiece, o[0]);
        step(o[1], g, 2 * i + 2, base + ROWS_STEP * (i + 1));
      }
    }
  }

  // the four wavefronts' sums, one after another
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
  float top[MT], f[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    top[m] = w_b[0][16 * m + c16];
#pragma unroll
    for (int w = 1; w < ROWS_WAVES; ++w) top[m] = __builtin_fmaxf(top[m], w_b[w][16 * m + c16]);
    f[m] = __builtin_amdgcn_exp2f(b[m] - top[m]);
  }
#pragma unroll 1
  for (int w = 0; w < ROWS_WAVES; ++w) {
    if (w == wave) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float* p = o_sum + (16 * m + c16) * PITCH + (4 * g4 + i) * N;
#pragma unroll
          for (int n = 0; n < N; ++n) p[n] = (w ? p[n] : 0.f) + acc[m][n][i] * f[m];
        }
    }
    __syncthreads();
  }

  // alone: the result; otherwise its part for kv8_attn_join
  KTIR_G(float)* ws = (KTIR_G(float)*)d.ws + blockIdx.x * PART<J, MT>;
  for (int at = threadIdx.x; at < TM; at += 256) {
    float bt = w_b[0][at], lt = 0.f;
    for (int w = 1; w < ROWS_WAVES; ++w) bt = __builtin_fmaxf(bt, w_b[w][at]);
    for (int w = 0; w < ROWS_WAVES; ++w) lt += w_l[w][at] * __builtin_amdgcn_exp2f(w_b[w][at] - bt);
    w_b[0][at] = bt;
    w_l[0][at] = lt;
    if (active > 1) {
      ws[TM * 64 * J + at] = bt;
      ws[TM * 64 * J + TM + at] = lt;
    } else if (d.lse && at < t.rows) {
      const int r = t.row0 + at;
      int a, z;
      seen(d, t, r, grp, &a, &z);
      ((KTIR_G(float)*)d.lse)[(t.q.start + r / grp) * d.lse_tok + (head * grp + r % grp) * d.lse_head] =
          a >= z ? -__builtin_inff() : (bt + 16.f + __builtin_amdgcn_logf(lt)) * 0.69314718055994530942f;
    }
  }
  __syncthreads();
  for (int at = threadIdx.x; at < t.rows * 16 * J; at += 256) {
    const int row = at / (16 * J), x4 = at % (16 * J) * 4;
    const f32x4_t o = *(const f32x4_t*)(o_sum + row * PITCH + x4);
    if (active > 1) {
      *(KTIR_G(f32x4_t)*)(ws + row * 64 * J + x4) = o;
      continue;
    }
    if (x4 >= D) continue;
    const int r = t.row0 + row;
    int a, z;
    seen(d, t, r, grp, &a, &z);
    const float inv = L_UNIT / w_l[0][row];
    const int64_t e = (t.q.start + r / grp) * d.out.tok + (head * grp + r % grp) * d.out.head + x4;
#pragma unroll
    for (int i = 0; i < 4; ++i) store_elem(d.out.ptr, e + i, d.dtype, a >= z ? 0.f : o[i] * inv);
  }
}

// The parts of a tile's splits, joined in their order: one wavefront per row, J columns a lane.
template <int J, int MT>
__global__ __launch_bounds__(256) void kv8_attn_join(const ktir_kv8_attn_t d, int* err) {
  constexpr int TM = 16 * MT, QUANT = ROWS_STEP * ROWS_WAVES;
  const ktir_kv8_t& c = d.cache;
  const int l = threadIdx.x & 63, grp = (int)(d.q_heads / c.heads), D = (int)c.columns, splits = d.splits;
  const int64_t item = blockIdx.x, head = item % c.heads, slot = item / c.heads;
  const Tile t = tile_of(d, slot, TM, grp, err);
  const int row = uni((int)(blockIdx.y * 4 + (threadIdx.x >> 6)));
  if (row >= t.rows) return;
  const int from = t.lo & ~(ROWS_STEP - 1), span = t.hi > from ? t.hi - from : 0;
  const int part = ((span + splits - 1) / splits + QUANT - 1) / QUANT * QUANT, active = span ? (span + part - 1) / part : 1;
  if (active <= 1) return;
  const KTIR_G(float)* ws = (const KTIR_G(float)*)d.ws + item * splits * PART<J, MT>;
  float top = B_NONE;
  for (int s = l; s < active; s += 64) top = __builtin_fmaxf(top, ws[s * PART<J, MT> + TM * 64 * J + row]);
  for (int o = 32; o; o >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o));
  float acc[J] = {}, lt = 0.f;
  for (int s = 0; s < active; ++s) {
    const KTIR_G(float)* p = ws + s * PART<J, MT>;
    const float f = __builtin_amdgcn_exp2f(p[TM * 64 * J + row] - top);
    lt += p[TM * 64 * J + TM + row] * f;
#pragma unroll
    for (int j = 0; j < J; ++j) acc[j] += p[row * 64 * J + 64 * j + l] * f;
  }
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
  s->part = TM * (64 * s->J + 2);
  // splits: enough workgroups for 256 CUs, no fewer than 256 keys each
  const int64_t items = s->slots * d.cache.heads, most = (d.max_k + 255) / 256;
  int64_t n = items ? 1024 / items : 1;
  n = n > most ? most : n;
  s->splits = n < 1 ? 1 : n > 64 ? 64 : (int)n;
}

template <int CODE, int J, int MT>
static int launch(const ktir_kv8_attn_t& d, const KV8Shape& s) {
  const int64_t items = s.slots * d.cache.heads, splits = d.splits < 1 ? 1 : d.splits;
  const hipStream_t st = stream_of(d.stream);
  hipLaunchKernelGGL((kv8_attn_rows<CODE, J, MT>), dim3((unsigned)(items * splits)), dim3(256), 0, st, d, device_error_flag());
  if (splits > 1)
    hipLaunchKernelGGL((kv8_attn_join<J, MT>), dim3((unsigned)items, 4 * MT), dim3(256), 0, st, d, device_error_flag());
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}

template <int CODE, int J>
static int launch_j(const ktir_kv8_attn_t& d, const KV8Shape& s) {
  return s.MT == 1 ? launch<CODE, J, 1>(d, s) : launch<CODE, J, 2>(d, s);
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
