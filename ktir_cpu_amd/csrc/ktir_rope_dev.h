// Device helpers of the rotary positions: angles, and vectors of pairs loaded, turned and stored.
#pragma once
#include "ktir_serve.h"

namespace ktir {

typedef float f4_t __attribute__((ext_vector_type(4)));

// cosine and sine of a pair at a position, times the amplitude, rounded once.  The angle passes
// 2^20 radians at far positions, where f32 holds it to a sixteenth: all of it is f64
// (the vector pipe's f64 and f32 instructions take as long).
__device__ __forceinline__ void rope_angle_of(int64_t pos, double freq, double amplitude, bool inverse, float* c, float* s) {
  double turns = (double)pos * freq * 0.15915494309189533577;
  turns -= rint(turns);
  double sn, cs;
  sincospi(2.0 * turns, &sn, &cs);
  *c = (float)(cs * amplitude);
  *s = (float)(inverse ? -(sn * amplitude) : sn * amplitude);
}
__device__ __forceinline__ void rope_angle(const ktir_rope_t& d, int64_t pos, int i, float* c, float* s) {
  rope_angle_of(pos, ((const KTIR_G(double)*)d.freq)[i], d.amplitude, d.inverse, c, s);
}

template <class D>
__device__ __forceinline__ int64_t rope_pos(const D& d, int64_t t) {
  return d.pos_dtype == KTIR_I64 ? ((const KTIR_G(int64_t)*)d.pos)[t] : (int64_t)ints(d.pos)[t];
}

// V pairs: 2 V values as f32, and back.  Half layout: V values at `a` and their V
// partners at `b`; interleaved: 2 V values from `a` on (b = a + V).
template <int DT, int V>
struct RopeRaw {
  uint32_t w[2][DT == KTIR_F32 ? V : (V + 1) / 2];
};

template <int DT, int V, bool PAST>
__device__ __forceinline__ void rope_load(uint64_t ptr, int64_t a, int64_t b, RopeRaw<DT, V>& r) {
  const int64_t e[2] = {a, b};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (V == 1) {
      if constexpr (DT == KTIR_F32) r.w[i][0] = ((const KTIR_G(uint32_t)*)ptr)[e[i]];
      else r.w[i][0] = ((const KTIR_G(uint16_t)*)ptr)[e[i]];
    } else {
      const KTIR_G(u4_t)* p = (const KTIR_G(u4_t)*)(ptr + e[i] * (DT == KTIR_F32 ? 4 : 2));
      const u4_t x = PAST ? __builtin_nontemporal_load(p) : *p;
#pragma unroll
      for (int k = 0; k < 4; ++k) r.w[i][k] = x[k];
    }
  }
}

template <int DT, int V>
__device__ __forceinline__ void rope_store(uint64_t ptr, int64_t a, int64_t b, const RopeRaw<DT, V>& r, bool two) {
  const int64_t e[2] = {a, b};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (i && !two) break;
    if constexpr (V == 1) {
      if constexpr (DT == KTIR_F32) ((KTIR_G(uint32_t)*)ptr)[e[i]] = r.w[i][0];
      else ((KTIR_G(uint16_t)*)ptr)[e[i]] = (uint16_t)r.w[i][0];
    } else {
      *(KTIR_G(u4_t)*)(ptr + e[i] * (DT == KTIR_F32 ? 4 : 2)) = u4_t{r.w[i][0], r.w[i][1], r.w[i][2], r.w[i][3]};
    }
  }
}

template <int DT>
__device__ __forceinline__ float rope_get(const uint32_t* w, int k) {
  if constexpr (DT == KTIR_F32) return __uint_as_float(w[k]);
  else {
    const uint32_t h = (w[k >> 1] >> (16 * (k & 1))) & 0xffffu;
    if constexpr (DT == KTIR_BF16) return __uint_as_float(h << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
  }
}

template <int DT>
__device__ __forceinline__ uint32_t rope_bits(float x) {
  if constexpr (DT == KTIR_F32) return __float_as_uint(x);
  else if constexpr (DT == KTIR_BF16) return __builtin_bit_cast(uint16_t, (__bf16)x);
  else return __builtin_bit_cast(uint16_t, (_Float16)x);
}

// x0 c - x1 s and x1 c + x0 s of V pairs
template <int DT, bool INTER, int V>
__device__ __forceinline__ void rope_turn_raw(RopeRaw<DT, V>& r, const float* c, const float* s) {
  float out[2][V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    float x, y;
    if constexpr (INTER && V > 1) {
      x = rope_get<DT>(r.w[2 * k / V], 2 * k % V);
      y = rope_get<DT>(r.w[(2 * k + 1) / V], (2 * k + 1) % V);
    } else {
      x = rope_get<DT>(r.w[0], k);
      y = rope_get<DT>(r.w[1], k);
    }
    const float u = __fsub_rn(__fmul_rn(x, c[k]), __fmul_rn(y, s[k])), v = __fadd_rn(__fmul_rn(y, c[k]), __fmul_rn(x, s[k]));
    if constexpr (INTER && V > 1) {
      out[2 * k / V][2 * k % V] = u;
      out[(2 * k + 1) / V][(2 * k + 1) % V] = v;
    } else {
      out[0][k] = u;
      out[1][k] = v;
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if constexpr (DT == KTIR_F32) r.w[i][k] = rope_bits<DT>(out[i][k]);
      else if constexpr (V == 1) r.w[i][0] = rope_bits<DT>(out[i][0]);
      else if (!(k & 1)) r.w[i][k / 2] = rope_bits<DT>(out[i][k]) | rope_bits<DT>(out[i][k + 1]) << 16;
    }
}

// A unit of columns: V pairs, or 2 V of the columns behind rot, as two vectors.
template <bool INTER, int V>
__device__ __forceinline__ void rope_columns(int u, int pairs, int half, int rot, int* a, int* b) {
  if (u < pairs) {
    *a = INTER ? 2 * u * V : u * V;
    *b = INTER ? *a + V : *a + half;
  } else {
    *a = rot + (u - pairs) * 2 * V;
    *b = *a + V;
  }
}

}  // namespace ktir
