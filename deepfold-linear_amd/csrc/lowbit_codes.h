// Codes of the few-bit caches (include/dfl_lowbit.h): 8 elements of a row a lane, so that a group of 32 is a quad of
// neighbouring lanes.  Every step is exact but the rounding to a code: multiplications by powers of two, the
// conversions of gfx950 between fp32 / bf16 and pairs of 4-bit elements with a power of two as their scale (round to nearest
// even, beyond 6 to 6).  The group's power of two keeps half a step everywhere: it is the lowest at which the largest
// magnitude rounds to a code, 7 steps and a half of the 4-bit grid's last interval [4, 6] or 127.5 of the integers.
#pragma once
#include "common.h"

namespace dfl {

constexpr int LB_GROUP = 32;
constexpr unsigned LB_NAN = 255;  // exponent byte of a group with an infinity or NaN

__host__ __device__ inline int lb_groups(int d) { return (d + LB_GROUP - 1) / LB_GROUP; }
__device__ __forceinline__ float lb_scale(unsigned e) { return __uint_as_float(e << 23); }

// The quad's exponent byte and this lane's 8 codes; all four lanes of a quad are active.
template <int BITS> __device__ __forceinline__ unsigned lb_encode(const float (&x)[8], unsigned (&w)[BITS / 4]) {
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0xb1, 0xf, 0xf, false));  // quad_perm 1,0,3,2
  top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x4e, 0xf, 0xf, false));  // quad_perm 2,3,0,1
  const int e0 = (int)(top >> 23);
  const unsigned m = top & 0x7fffffu;
  const bool up = (BITS == 4 ? m > 0x600000u : m >= 0x7f0000u) & (e0 < 254);
  const int e = max(e0 - (BITS == 4 ? 2 : 6) + (int)up, 1);
  const bool fine = e0 < 255;
  if constexpr (BITS == 4) {
    const float s = lb_scale(e);
    unsigned c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], s, 3);
    w[0] = fine ? c : 0u;
  } else {
    const float inv = lb_scale(254 - min(e, 253));
    unsigned u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // 1.5 * 2^23 + y: y rounded to the nearest even integer, two's complement in the low bits
      const float y = __builtin_amdgcn_fmed3f(x[i] * inv, -127.f, 127.f) + 12582912.f;
      u[i] = __float_as_uint(y);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned lo = __builtin_amdgcn_perm(u[4 * h + 1], u[4 * h], 0x0c0c0400u);
      const unsigned hi = __builtin_amdgcn_perm(u[4 * h + 3], u[4 * h + 2], 0x04000c0cu);
      w[h] = fine ? (lo | hi) : 0u;
    }
  }
  return fine ? (unsigned)e : LB_NAN;
}

// 8 values of a lane's codes; NaN where the byte says so.
template <int BITS> __device__ __forceinline__ void lb_decode(const unsigned (&w)[BITS / 4], unsigned e, float (&x)[8]) {
  const float s = e == LB_NAN ? __builtin_nanf("") : lb_scale(e);
  if constexpr (BITS == 4) {
    typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2;
    const float one = 1.f;
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], one, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], one, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], one, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], one, 3);
    x[0] = a[0] * s, x[1] = a[1] * s, x[2] = b[0] * s, x[3] = b[1] * s;
    x[4] = c[0] * s, x[5] = c[1] * s, x[6] = d[0] * s, x[7] = d[1] * s;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)(int8_t)(w[i / 4] >> (8 * (i % 4))) * s;
  }
}

// Elements 8 c .. 8 c + 7 of a row of d in fp32, zeros from d on.  FAST: 16-byte aligned rows and d a multiple of 8.
template <typename T, bool FAST> __device__ __forceinline__ void load8(const T* row, int c, int d, float (&x)[8]) {
  if (FAST) {
    typedef __attribute__((__vector_size__(4 * sizeof(unsigned)))) unsigned u4;
    constexpr int PARTS = (int)sizeof(T) / 2;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
    if (c * 8 >= d) return;
    u4 u[PARTS];
#pragma unroll
    for (int i = 0; i < PARTS; ++i) u[i] = reinterpret_cast<const u4*>(row + c * 8)[i];
    T e[8];
    __builtin_memcpy(e, u, sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = c * 8 + i < d ? to_f32(row[c * 8 + i]) : 0.f;
  }
}
// The same for 8 results.
template <typename T, bool FAST> __device__ __forceinline__ void store8(T* row, int c, int d, const float (&x)[8]) {
  if (FAST) {
    typedef __attribute__((__vector_size__(4 * sizeof(unsigned)))) unsigned u4;
    constexpr int PARTS = (int)sizeof(T) / 2;
    if (c * 8 >= d) return;
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x[i]);
    u4 u[PARTS];
    __builtin_memcpy(u, e, sizeof(e));
#pragma unroll
    for (int i = 0; i < PARTS; ++i) reinterpret_cast<u4*>(row + c * 8)[i] = u[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c * 8 + i < d) row[c * 8 + i] = from_f32<T>(x[i]);
  }
}

}  // namespace dfl
