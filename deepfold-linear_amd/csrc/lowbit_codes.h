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

// 8 elements of a row: as they lie in memory in bf16 (pairs), or in fp32.
template <typename T> struct Eight;
template <> struct Eight<bf16> {
  unsigned p[4];
};
template <> struct Eight<float> {
  float x[8];
};
// Elements 8 c .. 8 c + 7 of a row of d, zeros from d on.  FAST: 16-byte aligned rows and d a multiple of 8.
template <bool FAST> __device__ __forceinline__ void load8(Eight<bf16>& e, const bf16* row, int c, int d) {
  if (FAST) {
    const uint4 u = c * 8 < d ? *reinterpret_cast<const uint4*>(row + c * 8) : make_uint4(0u, 0u, 0u, 0u);
    e.p[0] = u.x, e.p[1] = u.y, e.p[2] = u.z, e.p[3] = u.w;
  } else {
    const unsigned short* at = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned lo = c * 8 + 2 * i < d ? at[c * 8 + 2 * i] : 0, hi = c * 8 + 2 * i + 1 < d ? at[c * 8 + 2 * i + 1] : 0;
      e.p[i] = lo | hi << 16;
    }
  }
}
template <bool FAST> __device__ __forceinline__ void load8(Eight<float>& e, const float* row, int c, int d) {
  if (FAST) {
    // (vectors of the language: of two float4 objects to choose from the compiler loads each element by itself)
    typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f4;
    f4 u = {}, v = {};
    if (c * 8 < d) u = reinterpret_cast<const f4*>(row + c * 8)[0], v = reinterpret_cast<const f4*>(row + c * 8)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) e.x[i] = u[i], e.x[4 + i] = v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) e.x[i] = c * 8 + i < d ? row[c * 8 + i] : 0.f;
  }
}
__device__ __forceinline__ unsigned quad_max(unsigned x) {
  x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, false));     // quad_perm 1,0,3,2
  return max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, false));  // quad_perm 2,3,0,1
}
// Largest magnitude of the quad, as the upper half of an fp32 number's bits (bf16), or all of them.
__device__ __forceinline__ unsigned lb_top(const Eight<bf16>& e) {
  typedef __attribute__((__vector_size__(2 * sizeof(unsigned short)))) unsigned short pair;
  pair m = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned a = e.p[i] & 0x7fff7fffu;
    pair x;
    __builtin_memcpy(&x, &a, 4);
    m = __builtin_elementwise_max(m, x);
  }
  return quad_max(max((unsigned)m[0], (unsigned)m[1])) << 16;
}
__device__ __forceinline__ unsigned lb_top(const Eight<float>& e) {
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(e.x[i]) & 0x7fffffffu);
  return quad_max(top);
}
__device__ __forceinline__ unsigned lb_fp4(const Eight<bf16>& e, float s) {
  typedef __attribute__((__vector_size__(2 * sizeof(bf16)))) bf16 pair;
  pair x[4];
  __builtin_memcpy(x, e.p, 16);
  unsigned c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, x[0], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, x[1], s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, x[2], s, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, x[3], s, 3);
}
__device__ __forceinline__ unsigned lb_fp4(const Eight<float>& e, float s) {
  unsigned c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, e.x[0], e.x[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, e.x[2], e.x[3], s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, e.x[4], e.x[5], s, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, e.x[6], e.x[7], s, 3);
}
__device__ __forceinline__ void lb_floats(const Eight<bf16>& e, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(e.p[i] << 16), x[2 * i + 1] = __uint_as_float(e.p[i] & 0xffff0000u);
}
__device__ __forceinline__ void lb_floats(const Eight<float>& e, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = e.x[i];
}
// The low bytes of four words.
__device__ __forceinline__ unsigned low_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __builtin_amdgcn_perm(b, a, 0x0c0c0400u) | __builtin_amdgcn_perm(d, c, 0x04000c0cu);
}

// The quad's exponent byte and this lane's 8 codes; all four lanes of a quad are active.
template <int BITS, typename T> __device__ __forceinline__ unsigned lb_encode(const Eight<T>& v, unsigned (&w)[BITS / 4]) {
  const unsigned top = lb_top(v), m = top & 0x7fffffu;
  const int e0 = (int)(top >> 23);
  const bool up = (BITS == 4 ? m > 0x600000u : m >= 0x7f0000u) & (e0 < 254), fine = e0 < 255;
  const int e = max(e0 - (BITS == 4 ? 2 : 6) + (int)up, 1);
  if constexpr (BITS == 4) {
    w[0] = fine ? lb_fp4(v, lb_scale(e)) : 0u;
  } else {
    const float inv = lb_scale(254 - min(e, 253));
    float x[8];
    unsigned u[8];
    lb_floats(v, x);
    // 1.5 * 2^23 + x / step: rounded to the nearest even integer, two's complement in the low bits
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(__builtin_fmaf(x[i], inv, 12582912.f));
    if (e0 == 254) {  // the only groups that reach beyond 127.5 steps
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(__builtin_amdgcn_fmed3f(x[i] * inv, -127.f, 127.f) + 12582912.f);
    }
    w[0] = fine ? low_bytes(u[0], u[1], u[2], u[3]) : 0u;
    w[1] = fine ? low_bytes(u[4], u[5], u[6], u[7]) : 0u;
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
