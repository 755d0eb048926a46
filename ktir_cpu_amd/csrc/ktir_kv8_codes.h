// Device helpers of what writes the 8-bit cache: values as codes of a page's scale, and back.
#pragma once
#include "ktir_serve.h"

namespace ktir {

constexpr float LEAST_SCALE = 0x1p-100f;     // codes of a page of zeros are zeros times this

template <int CODE>
constexpr float PER_TOP = 1.f / (CODE == KTIR_I8 ? 127.f : 448.f);

// four values over their scale as codes; NAN_TOO: some may be NaN, and stay so (the clamp makes a bound of one)
template <int CODE, bool NAN_TOO = false>
__device__ __forceinline__ uint32_t codes4(const float* x) {
  if constexpr (CODE == KTIR_I8) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = (int)__builtin_amdgcn_fmed3f(__builtin_rintf(x[i]), -127.f, 127.f);
      w |= (uint32_t)(c & 0xff) << (8 * i);
    }
    return w;
  } else {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[i] = __builtin_amdgcn_fmed3f(x[i], -448.f, 448.f);
      if (NAN_TOO) y[i] = x[i] != x[i] ? x[i] : y[i];
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
  }
}

template <int CODE>
__device__ __forceinline__ void values4(uint32_t w, float* x) {
  if constexpr (CODE == KTIR_I8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
  } else {
    x[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0);
    x[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
    x[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2);
    x[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
  }
}

// 16 new values: packed as they are, and as f32 times `f`
struct New16 {
  uint32_t w[8];
};

__device__ __forceinline__ New16 new16(uint64_t ptr, int64_t e, bool wide) {
  New16 r;
  const KTIR_G(uint16_t)* p = (const KTIR_G(uint16_t)*)ptr + e;
  if (wide) {
    const u4_t a = ((const KTIR_G(u4_t)*)p)[0], b = ((const KTIR_G(u4_t)*)p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = a[i], r.w[4 + i] = b[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
  }
  return r;
}

template <bool BF16>
__device__ __forceinline__ u4_t codes16(const New16& x, float f, int code) {
  u4_t o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t w = x.w[2 * i + k];
      if constexpr (BF16) {
        v[2 * k] = __uint_as_float(w << 16) * f;
        v[2 * k + 1] = __uint_as_float(w & 0xffff0000u) * f;
      } else {
        v[2 * k] = (float)__builtin_bit_cast(_Float16, (uint16_t)w) * f;
        v[2 * k + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16)) * f;
      }
    }
    o[i] = code == KTIR_I8 ? codes4<KTIR_I8>(v) : codes4<KTIR_E4M3>(v);
  }
  return o;
}

// the largest of 16 packed absolute values: of both types the bits grow with the value, and past infinity for NaN
__device__ __forceinline__ uint32_t top16(const New16& x, uint32_t top) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = x.w[i] & 0x7fffu, b = (x.w[i] >> 16) & 0x7fffu;
    top = top > a ? top : a;
    top = top > b ? top : b;
  }
  return top;
}

}  // namespace ktir
