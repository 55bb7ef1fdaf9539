// One token's attention over a rolling cache in 8 or 4 bits.
//
// Codes become bf16 operands of 16x16x32 matrix instructions in registers, exactly (a code has at most 7 bits, its scale
// is a power of two), straight from the loads: no LDS between.  In vector instructions alone the products of four heads
// would take longer than the codes take to arrive.  A wave takes 32 slots at a time:
//   scores (slots x heads): A = 16 rows of keys, lane l one row and a quarter l / 16 of its elements, as they lie in
//     memory; B = the queries with the same elements.  Rows are taken such that lane l of the accumulator has head l % 16
//     and the slots 4 r + l / 16, r = 0 .. 3, of a half block.
//   outputs (heads x columns): A = the weights, head l % 16, slots 4 r + l / 16 of both halves: they stay in their lane;
//     B = 16 columns of the values of these slots: lane l loads the elements l % 16 * DP / 16 .. of each of its slots, so
//     that a load of the wave has four neighbouring rows.
// The 16 rows of the weights hold GP heads in TERMS parts: bf16 results take two bf16 numbers for a weight (16 bits of
// it), fp32 results three (24 bits), so no weight is rounded to 8 bits and the matrix rows would be idle otherwise.  fp32
// queries are three bf16 numbers, products of their own.  Sums, references and outputs are fp32.
//
// Bounds: the cache's bytes, and about 230 vector instructions a block of 4 bits.  Kernels in a trace: 32 sequences of 4100
// slots, 32 / 8 heads, d 128, 4 bits, 143 MB: 28.9 us, 4.9 TB/s of the 6.2 that a copy reaches (bf16 caches, 537 MB: 106 us).
// One sequence of 131072 slots, the same heads, 8 bits, 276 MB: 47-48 us, 5.8 TB/s, and 4.1-4.6 us for joining the splits.
// One sequence of 1028 slots, 16 / 4 heads, d 64, 4 bits: 9.3 us, latency.
// Registers: the keys' are free for the next block once the scores are formed, the values' once the outputs are, so that one
// set lets three waves a SIMD run (two sets, two waves: 33.7 us); loads go through buffer resources (with 64-bit addresses a
// lane and clamped rows 36 us).
#include "lowbit_args.h"
#include "lowbit_codes.h"
#include "window_engine.h"

#include <algorithm>

namespace dfl {

template <typename T> struct LbHeads {
  static constexpr int TERMS = sizeof(T) == 2 ? 2 : 4;  // parts of a weight (the fourth of fp32 is zero)
  static constexpr int GP = 16 / TERMS;                 // heads of a tile
  static constexpr int QT = sizeof(T) == 2 ? 1 : 3;     // parts of a query
};
// Waves a SIMD that the registers let run without spilling, and so the largest workgroup: one a CU.
constexpr int lb_waves(int size, int DP, int NT) {
  return DP < 128 ? (NT == 2 ? 2 : 3) : NT == 2 ? (size == 4 ? 1 : 2) : (size == 4 ? 2 : 3);
}
// Small workgroups overlap on a CU (lowbit_decode_plan): of bf16 rows of at most 64 elements the registers are held down to
// four waves a SIMD (64 x 16 / 16 heads of 2052 slots, 4 bits 51 us with three).
constexpr int lb_least_waves(int size, int DP, int NT) { return size == 2 && DP < 128 && NT == 1 ? 4 : lb_waves(size, DP, NT); }
// A reference is moved when a score passes it by more than this: weights stay below 2^8.
constexpr float LB_LAZY = 8.f;
// With S <= 2^c slots, sums of weights times values stay below 2^126 as long as the values' exponents lie below 239 - c (a
// code has 7 bits).  A wave that has met a higher one goes through its slots again with a reference c + 10 above the largest
// score: values below 2^128 then make no more of a sum either, and the join needs to know nothing of it.  (Weights below
// 2^(c - 116) of the largest vanish there.)
__device__ __forceinline__ int lb_lift(int S) { return 42 - __clz(S - 1); }
__device__ __forceinline__ unsigned lb_high(int S) { return 249u - lb_lift(S); }
constexpr long long CUS = 256;

// Distance of the token, `rest` slots behind the first one of the window, to the position that slot s in use holds.
__device__ __forceinline__ int lb_distance(int s, int t, int n_sink, int window, int rest) {
  const int back = rest - (s - n_sink);
  return s < n_sink ? t - s : back + (back < 0 ? window : 0);
}
// Upper halves: exact where the values have 8 bits, else cut off.
__device__ __forceinline__ unsigned bf16_pair(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

// Two neighbouring 4-bit elements (byte I of w) as a bf16 pair.
template <int I> __device__ __forceinline__ unsigned fp4_pair(unsigned w, float s) {
  const auto p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, I);
  unsigned u;
  __builtin_memcpy(&u, &p, 4);
  return u;
}
template <int I> __device__ __forceinline__ float int8_at(unsigned w, float s) { return (float)(int8_t)(w >> (8 * I)) * s; }

typedef __amdgpu_buffer_rsrc_t lb_rsrc;
// `bytes` bytes from p on; loads behind them give zero.
__device__ __forceinline__ lb_rsrc lb_buffer(const uint8_t* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, bytes, 0x00020000);
}
// N bytes at lane + row.  LB_ONCE: not kept in the caches (the values; 8 bits, one sequence of 131072 slots 54.7 -> 48.5 us,
// with the keys too 50.9; 4 bits, 32 sequences of 4100 31.5 -> 31.0).
constexpr int LB_ONCE = 2;
template <int N, int AUX = 0, int W>
__device__ __forceinline__ void lb_load(unsigned (&w)[W], lb_rsrc b, unsigned lane, unsigned row) {
  static_assert(W == (N + 3) / 4, "whole dwords");
  if constexpr (N == 1) w[0] = __builtin_amdgcn_raw_buffer_load_b8(b, lane, row, AUX);
  else if constexpr (N == 2) w[0] = __builtin_amdgcn_raw_buffer_load_b16(b, lane, row, AUX);
  else if constexpr (N == 4) w[0] = __builtin_amdgcn_raw_buffer_load_b32(b, lane, row, AUX);
  else if constexpr (N == 8) {
    const auto x = __builtin_amdgcn_raw_buffer_load_b64(b, lane, row, AUX);
    w[0] = x[0], w[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N / 16; ++i) {
      const auto x = __builtin_amdgcn_raw_buffer_load_b128(b, lane + 16 * i, row, AUX);
      w[4 * i] = x[0], w[4 * i + 1] = x[1], w[4 * i + 2] = x[2], w[4 * i + 3] = x[3];
    }
  }
}

union LbFrag {
  unsigned u[4];
  bf16x8 v;
};

template <typename T, int BITS, int DP, int NT, bool REL>
__global__ void __launch_bounds__(256 * lb_waves(sizeof(T), DP, NT), lb_least_waves(sizeof(T), DP, NT))
    lowbit_decode_kernel(LowbitDecodeArgs a) {
  using Hd = LbHeads<T>;
  constexpr int GP = Hd::GP, QT = Hd::QT, GB = NT * GP;
  constexpr int KF = DP / 32;            // matrix instructions of a score tile; fragments of a lane's quarter row
  constexpr int KW = DP * BITS / 128;    // dwords of a lane's quarter row: KF of 4 bits, 2 KF of 8
  constexpr int NC = DP / 16;            // columns of a lane
  constexpr int VB = NC * BITS / 8;      // bytes of them: 1, 2, 4 or 2, 4, 8
  constexpr int VW = (VB + 3) / 4;
  extern __shared__ __align__(16) unsigned char smem[];
  const int waves = blockDim.x >> 6;
  float* s_ml = reinterpret_cast<float*>(smem);  // [waves][GB][2]
  float* s_o = s_ml + waves * GB * 2;            // [waves][GB][DP]
  uint8_t* s_own = reinterpret_cast<uint8_t*>(s_o + waves * GB * DP);  // [2][DP * BITS / 8] the token's own codes
  uint8_t* s_exp = s_own + 2 * DP * BITS / 8;                      // [2][4]
  float* s_tab = reinterpret_cast<float*>(s_exp + 8);              // [GB][buckets]
  uint8_t* s_lut = reinterpret_cast<uint8_t*>(s_tab + (REL ? GB * a.rel.buckets() : 0));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, h = lane >> 4;
  const int G = a.H / a.Hk, nhg = (G + GB - 1) / GB;
  int x = blockIdx.x;
  const int sp = x % a.n_split;
  x /= a.n_split;
  const int hg = x % nhg, bh = x / nhg, b = bh / a.Hk, hk = bh % a.Hk;
  const int g0 = hg * GB, gn = min(GB, G - g0), h0 = hk * G + g0;
  const int t = a.lengths[b], S = a.n_sink + a.window;
  const int used = t < 0 ? 0 : (t >= S ? S : t + 1);
  const int own = t < a.n_sink ? t : a.n_sink + (t - a.n_sink) % a.window;  // the token's own slot
  const int begin = sp * a.chunk, end = min(used, begin + a.chunk);
  const bool mine = t >= 0 && own >= begin && own < end;
  const int groups = lb_groups(a.d), nch = 4 * groups;

  const uint8_t* kc = a.kc.codes + b * a.kc.sb + hk * a.kc.sh;
  const uint8_t* vc = a.vc.codes + b * a.vc.sb + hk * a.vc.sh;
  const uint8_t* ke = a.kc.exps + b * a.kc.esb + hk * a.kc.esh;
  const uint8_t* ve = a.vc.exps + b * a.vc.esb + hk * a.vc.esh;

  const int kg = DP / 4 * h / 32, vg = n * NC / 32;   // groups of the lane's key and value elements
  const bool kin = kg < groups, vin = vg < groups;    // (96 of 128 elements: the last quarter has none)
  const int kge = min(kg, groups - 1), vge = min(vg, groups - 1);
  struct Raw {
    unsigned k[2][KW], v[8][VW];
    unsigned ke[2], ve[2][4];
  };
  // Loads through buffer resources: what the block and the row have in an address is scalar, a lane adds one register, and
  // what lies behind the last slot in use (or beside the row: 96 of 128 elements) is not read and counts as zero.  That needs
  // the scalar offset to count: gfx950 takes each dword of a raw buffer's load to be outside where lane and scalar offset
  // together pass the size, also where the scalar one does alone (tests/test_gpu_buffer_range.py holds it to that).  With the
  // row in the lane's offset wherever a block ends behind the last slot, or with a resource for each row, bf16 calls take 3
  // to 9 % longer.
  constexpr unsigned NOWHERE = 0x80000000u;  // (with any scalar offset, all below 2^31, neither inside nor past 2^32)
  const int kofs = h * (KW * 4), vofs = n * VB, ksn = (int)a.kc.sn, vsn = (int)a.vc.sn;
  const int kn = 4 * (n & 3) + (n >> 2);  // the slot of a half block that the lane's row of keys is
  const unsigned kat = kin ? kn * ksn + kofs : NOWHERE, vat = vin ? h * vsn + vofs : NOWHERE;
  const unsigned keat = kge * (unsigned)a.kc.esg + kn, veat = vge * (unsigned)a.vc.esg;
  const int S4 = (S + 3) & ~3;  // (a dword of exponents may reach behind the last slot)
  const auto kexp = lb_buffer(ke, (groups - 1) * (int)a.kc.esg + S4), vexp = lb_buffer(ve, (groups - 1) * (int)a.vc.esg + S4);
  Raw r;
  auto load_keys = [&](int s0) {
    const auto kb = lb_buffer(kc + s0 * a.kc.sn, min(32, end - s0) * ksn);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      lb_load<KW * 4>(r.k[u], kb, kat, 16 * u * ksn);
      r.ke[u] = __builtin_amdgcn_raw_buffer_load_b8(kexp, keat, s0 + 16 * u, 0);
    }
  };
  auto load_values = [&](int s0) {
    const auto vb = lb_buffer(vc + s0 * a.vc.sn, min(32, end - s0) * vsn);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      lb_load<16>(r.ve[u], vexp, veat, s0 + 16 * u);
#pragma unroll
      for (int j = 0; j < 4; ++j) lb_load<VB, LB_ONCE>(r.v[4 * u + j], vb, vat, (16 * u + 4 * j) * vsn);
    }
  };
  // the first block is on its way while the token and the queries are prepared
  const int first = begin + 32 * wave, stride = 32 * waves;
  if (first < end) load_keys(first), load_values(first);

  // The token's own codes: from the call's rows into LDS, and into the cache by one workgroup.
  if (mine && wave < 2 && lane < nch) {
    const T* row = wave ? reinterpret_cast<const T*>(a.v) + b * a.vsb + hk * a.vsh
                        : reinterpret_cast<const T*>(a.k) + b * a.ksb + hk * a.ksh;
    Eight<T> e;
    unsigned w[BITS / 4];
    load8<false>(e, row, lane, a.d);
    const unsigned ex = lb_encode<BITS>(e, w);
    unsigned* at = reinterpret_cast<unsigned*>(s_own + wave * (DP * BITS / 8) + lane * BITS);
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i) at[i] = w[i];
    if (lane % 4 == 0) s_exp[wave * 4 + lane / 4] = (uint8_t)ex;
    if (hg == 0) {
      const LowbitCache& c = wave ? a.vc : a.kc;
      unsigned* to = reinterpret_cast<unsigned*>(c.codes + b * c.sb + hk * c.sh + own * c.sn + lane * BITS);
#pragma unroll
      for (int i = 0; i < BITS / 4; ++i) to[i] = w[i];
      if (lane % 4 == 0) c.exps[b * c.esb + hk * c.esh + lane / 4 * c.esg + own] = (uint8_t)ex;
    }
  }
  if (REL) {
    const int nb = a.rel.buckets(), dist = a.rel.dist();
    for (int e = threadIdx.x; e < gn * nb; e += blockDim.x) s_tab[e] = a.table[(size_t)h0 * nb + e] * LOG2E;
    for (int e = threadIdx.x; e <= dist; e += blockDim.x) s_lut[e] = (uint8_t)rel_bucket(a.rel, -e);
  }
  // The queries: lane's column n is head n % GP of a tile, elements DP / 4 * h .. of it.  They take the scale's power of
  // two, which changes none of their digits, where it is below 1 (above, a query may have no room for it); the scores take
  // the rest of the scale.
  const float sc0 = a.scale * LOG2E, two = fminf(__uint_as_float(__float_as_uint(sc0) & 0x7f800000u), 1.f), sc = sc0 / two;
  LbFrag q[NT][QT][KF];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int g = i * GP + n % GP;
    const T* row = reinterpret_cast<const T*>(a.q) + b * a.qsb + (h0 + min(g, gn - 1)) * a.qsh;
#pragma unroll
    for (int f = 0; f < KF; ++f) {
      float x[8];
      if (a.q_fast) load8<T, true>(row, KF * h + f, a.d, x);
      else load8<T, false>(row, KF * h + f, a.d, x);
      // Parts cut off, not rounded: a finite query has no infinite part.  (x * two is a quiet NaN where x is one, and stays
      // one cut off.)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        float lo = x[e] * two, hi = x[e + 1] * two;
        const bool finite_lo = fabsf(lo) < INFINITY, finite_hi = fabsf(hi) < INFINITY;
#pragma unroll
        for (int p = 0; p < QT; ++p) {
          q[i][p][f].u[e / 2] = g < gn ? bf16_pair(lo, hi) : 0u;
          lo = finite_lo ? lo - __uint_as_float(__float_as_uint(lo) & 0xffff0000u) : 0.f;
          hi = finite_hi ? hi - __uint_as_float(__float_as_uint(hi) & 0xffff0000u) : 0.f;
        }
      }
    }
  }
  lds_barrier();  // (not __syncthreads, which would wait for the block's loads)

  const int term = n / GP;
  const float sel1 = term >= 1 ? -1.f : 0.f, sel2 = term >= 2 ? -1.f : 0.f;
  f32x4 o[NT][NC];
  float m[NT], l[NT];
  unsigned top = 0;  // the highest exponent in use
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    m[i] = NEG_BIG, l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) o[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  f32x4 none[2] = {};  // what the scores of a block start from
  float slack = LB_LAZY;
  auto step = [&](int s0) {
    if (mine && s0 <= own && own < s0 + 32) {  // the token's own slot, as its codes stand
      const int at = own - s0;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (16 * u + kn == at) {
          const unsigned* p = reinterpret_cast<const unsigned*>(s_own + (kin ? kofs : 0));
#pragma unroll
          for (int i = 0; i < KW; ++i) r.k[u][i] = p[i];
          r.ke[u] = s_exp[kge];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (16 * u + 4 * j + h == at) {
            const uint8_t* p = s_own + DP * BITS / 8 + (vin ? vofs : 0);
            if constexpr (VB == 1) r.v[4 * u + j][0] = *p;
            else if constexpr (VB == 2) r.v[4 * u + j][0] = *reinterpret_cast<const unsigned short*>(p);
            else
#pragma unroll
              for (int i = 0; i < VW; ++i) r.v[4 * u + j][i] = reinterpret_cast<const unsigned*>(p)[i];
            r.ve[u][j] = (unsigned)s_exp[4 + vge] << (8 * h);
          }
      }
    }
    if (s0 + 32 > end) {  // the wave's last block: slots that are not in use score -inf, their exponents are not looked at
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (s0 + 16 * u + kn >= end) r.ke[u] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool in = s0 + 16 * u + 4 * j + h < end;
          none[u][j] = in ? 0.f : -INFINITY;
          if (!in) r.ve[u][j] = 0;
        }
      }
    }
    // scores
    f32x4 y[2][NT];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float ks = lb_scale(r.ke[u]);
      top = max(top, r.ke[u]);
#pragma unroll
      for (int i = 0; i < NT; ++i) y[u][i] = none[u];
#pragma unroll
      for (int f = 0; f < KF; ++f) {
        LbFrag k;
        if constexpr (BITS == 4) {
          const unsigned w = r.k[u][f];
          k.u[0] = fp4_pair<0>(w, ks), k.u[1] = fp4_pair<1>(w, ks), k.u[2] = fp4_pair<2>(w, ks), k.u[3] = fp4_pair<3>(w, ks);
        } else {
          const unsigned w0 = r.k[u][2 * f], w1 = r.k[u][2 * f + 1];
          k.u[0] = bf16_pair(int8_at<0>(w0, ks), int8_at<1>(w0, ks)), k.u[1] = bf16_pair(int8_at<2>(w0, ks), int8_at<3>(w0, ks));
          k.u[2] = bf16_pair(int8_at<0>(w1, ks), int8_at<1>(w1, ks)), k.u[3] = bf16_pair(int8_at<2>(w1, ks), int8_at<3>(w1, ks));
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int p = 0; p < QT; ++p)
            y[u][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k.v, q[i][p][f].v, y[u][i], 0, 0, 0);
      }
    }
    if (s0 + stride < end) load_keys(s0 + stride);
    // weights
    LbFrag w[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      float mx = NEG_BIG;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float v = y[u][i][j] * sc;
          if (REL) {
            const int at = min(s0 + 16 * u + 4 * j + h, end - 1);
            const int bk = s_lut[min(lb_distance(at, t, a.n_sink, a.window, own - a.n_sink), a.rel.dist())];
            v += s_tab[min(i * GP + n % GP, gn - 1) * a.rel.buckets() + bk];
          }
          y[u][i][j] = v;
          mx = fmaxf(mx, v);
        }
      if (__any(mx > m[i] + slack)) {
        mx = max_groups(fmaxf(mx + (LB_LAZY - slack), m[i]));
        const float al = fast_exp2(m[i] - mx);
        m[i] = mx;
        l[i] *= al;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float ar = __shfl(al, 4 * h + r, WAVE);
#pragma unroll
          for (int c = 0; c < NC; ++c) o[i][c][r] *= ar;
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[j] = fast_exp2(y[u][i][j] - m[i]);
          l[i] += p[j];
          // the part of the weight that this lane's row holds
          p[j] = __builtin_fmaf(sel1, (float)(bf16)p[j], p[j]);
          if constexpr (Hd::TERMS > 2) {
            p[j] = __builtin_fmaf(sel2, (float)(bf16)p[j], p[j]);
            if (term > 2) p[j] = 0.f;
          }
        }
        typedef __attribute__((__vector_size__(2 * sizeof(bf16)))) bf16 pair;
        const pair a0 = {(bf16)p[0], (bf16)p[1]}, a1 = {(bf16)p[2], (bf16)p[3]};
        __builtin_memcpy(&w[i].u[2 * u], &a0, 4);
        __builtin_memcpy(&w[i].u[2 * u + 1], &a1, 4);
      }
    }
    // outputs
    float vs[8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned e = __builtin_amdgcn_ubfe(r.ve[u][j], 8 * h, 8);
        top = max(top, e);
        vs[4 * u + j] = lb_scale(e);
      }
    }
    auto column = [&](int c, const LbFrag& v) {
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[i].v, v.v, o[i][c], 0, 0, 0);
    };
    if constexpr (BITS == 4) {
      auto two = [&](auto I) {
        constexpr int B = decltype(I)::value;
        if constexpr (2 * B < NC) {
          unsigned e[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] = fp4_pair<B>(r.v[j][0], vs[j]);
          LbFrag lo, hi;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            lo.u[j] = __builtin_amdgcn_perm(e[2 * j + 1], e[2 * j], 0x05040100u);
            hi.u[j] = __builtin_amdgcn_perm(e[2 * j + 1], e[2 * j], 0x07060302u);
          }
          column(2 * B, lo);
          column(2 * B + 1, hi);
        }
      };
      two(std::integral_constant<int, 0>{});
      two(std::integral_constant<int, 1>{});
      two(std::integral_constant<int, 2>{});
      two(std::integral_constant<int, 3>{});
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        LbFrag v;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v.u[j] = bf16_pair((float)(int8_t)(r.v[2 * j][c / 4] >> (8 * (c % 4))) * vs[2 * j],
                             (float)(int8_t)(r.v[2 * j + 1][c / 4] >> (8 * (c % 4))) * vs[2 * j + 1]);
        column(c, v);
      }
    }
  };
  for (;;) {
    // the next block's keys are loaded once this one's are used, its values likewise
    for (int s0 = first; s0 < end; s0 += stride) {
      step(s0);
      if (s0 + stride < end) load_values(s0 + stride);
    }
    if (slack != LB_LAZY || !__any(top >= lb_high(S)) || __any(top == LB_NAN)) break;
    slack = LB_LAZY - (float)lb_lift(S);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      m[i] = NEG_BIG, l[i] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) o[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    none[0] = none[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    load_keys(first), load_values(first);  // (top is not 0: the wave has slots)
  }

  // The waves' parts: weights' parts and lanes joined, then the waves in LDS.
  const bool poison = __any(top == LB_NAN);
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    float sum = sum_groups(l[i]);
    if (poison) sum = __builtin_nanf("");
    if (lane < GP) {
      s_ml[(wave * GB + i * GP + lane) * 2] = m[i];
      s_ml[(wave * GB + i * GP + lane) * 2 + 1] = sum;
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = o[i][c][r];  // row 4 h + r: head (4 h + r) % GP, part (4 h + r) / GP
        if constexpr (GP == 4) v = xor16_pair(v, false);
        v = xor32_pair(v, false);
        if (4 * h < GP) s_o[(wave * GB + i * GP + 4 * h + r) * DP + n * NC + c] = v;
      }
  }
  __syncthreads();
  // (A thread's columns: of many heads four, so that no thread does this twice: 16 x 16 / 1 heads of 8196 slots 18.6 -> 16.9 us;
  // of few one, 1 x 16 / 4 heads 9.2 and 9.4 with four.)
  constexpr int CW = NT == 2 ? 4 : 1;
  typedef __attribute__((__vector_size__(CW * sizeof(float)))) float cols;
  for (int e = threadIdx.x; e < gn * (DP / CW); e += blockDim.x) {
    const int g = e / (DP / CW), col = e % (DP / CW) * CW;
    float mx = NEG_BIG;
    for (int r = 0; r < waves; r += 4)  // (a multiple of 4)
#pragma unroll
      for (int k = 0; k < 4; ++k) mx = fmaxf(mx, s_ml[((r + k) * GB + g) * 2]);
    float sl = 0.f;
    cols so = {};
    for (int r = 0; r < waves; r += 4)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float al = fast_exp2(s_ml[((r + k) * GB + g) * 2] - mx);
        const cols v = *reinterpret_cast<const cols*>(s_o + ((r + k) * GB + g) * DP + col);
        sl = __builtin_fmaf(s_ml[((r + k) * GB + g) * 2 + 1], al, sl);
#pragma unroll
        for (int c = 0; c < CW; ++c) so[c] = __builtin_fmaf(v[c], al, so[c]);
      }
    const size_t head = (size_t)b * a.H + h0 + g;
    if (a.n_split == 1) {
      T* o = reinterpret_cast<T*>(a.o) + head * a.d + col;
#pragma unroll
      for (int c = 0; c < CW; ++c)
        if (col + c < a.d) o[c] = from_f32<T>(sl == 0.f ? 0.f : so[c] / sl);
    } else {
      float* part = a.part + (head * a.n_split + sp) * (DP + 2);
      if (col == 0) part[0] = mx, part[1] = sl;
#pragma unroll
      for (int c = 0; c < CW; ++c) part[2 + col + c] = so[c];
    }
  }
}

// The splits' outputs joined, in split order: a workgroup a head; their references and sums in LDS first, so that the
// loop over the outputs has only independent loads.
template <typename T, int DP> __global__ void __launch_bounds__(128) lowbit_join_kernel(LowbitDecodeArgs a) {
  extern __shared__ float s_w[];  // [n_split] weights
  const size_t head = blockIdx.x;
  const float* part = a.part + head * a.n_split * (DP + 2);
  float mx = NEG_BIG;
  for (int s = threadIdx.x; s < a.n_split; s += 128) mx = fmaxf(mx, s_w[s] = part[(size_t)s * (DP + 2)]);
  __shared__ float s_red[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int o = 32; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, WAVE));
  if (lane == 0) s_red[wave] = mx;
  __syncthreads();
  mx = fmaxf(s_red[0], s_red[1]);
  float l = 0.f;
  for (int s = threadIdx.x; s < a.n_split; s += 128) {
    s_w[s] = fast_exp2(s_w[s] - mx);
    l = __builtin_fmaf(s_w[s], part[(size_t)s * (DP + 2) + 1], l);
  }
  l = wave_sum(l);
  if (lane == 0) s_red[2 + wave] = l;
  __syncthreads();
  l = s_red[2] + s_red[3];
  const int col = threadIdx.x;
  if (col >= a.d) return;
  float o = 0.f;
  for (int s0 = 0; s0 < a.n_split; s0 += 8) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = s0 + k < a.n_split ? part[(size_t)(s0 + k) * (DP + 2) + 2 + col] : 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) o = __builtin_fmaf(v[k], s0 + k < a.n_split ? s_w[s0 + k] : 0.f, o);
  }
  reinterpret_cast<T*>(a.o)[head * a.d + col] = from_f32<T>(l == 0.f ? 0.f : o / l);
}

template <typename T, int BITS, int DP, int NT, bool REL> static hipError_t decode_l(const LowbitDecodeArgs& a, hipStream_t s) {
  constexpr int GB = NT * LbHeads<T>::GP;
  const int G = a.H / a.Hk, nhg = (G + GB - 1) / GB;
  const size_t lds = (size_t)a.waves * GB * (DP + 2) * 4 + 2 * DP * BITS / 8 + 8 +
                     (REL ? (size_t)GB * a.rel.buckets() * 4 + a.rel.dist() + 1 : 0);
  auto kern = lowbit_decode_kernel<T, BITS, DP, NT, REL>;
  hipError_t e = set_lds_limit((const void*)kern, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3((unsigned)(a.B * a.Hk * nhg * a.n_split)), dim3(64 * a.waves), lds, s, a);
  if ((e = hipGetLastError()) != hipSuccess || a.n_split == 1) return e;
  hipLaunchKernelGGL((lowbit_join_kernel<T, DP>), dim3((unsigned)(a.B * a.H)), dim3(128), a.n_split * 4, s, a);
  return hipGetLastError();
}
template <typename T, int BITS, int DP> static hipError_t decode_d(LowbitDecodeArgs a, hipStream_t s) {
  const long long size = sizeof(T);
  a.q_fast = a.d % 8 == 0 && (((uintptr_t)a.q | (uintptr_t)(a.qsb * size) | (uintptr_t)(a.qsh * size)) & 15) == 0;
  const bool two = a.H / a.Hk > LbHeads<T>::GP;
  if (a.table) return two ? decode_l<T, BITS, DP, 2, true>(a, s) : decode_l<T, BITS, DP, 1, true>(a, s);
  return two ? decode_l<T, BITS, DP, 2, false>(a, s) : decode_l<T, BITS, DP, 1, false>(a, s);
}
template <typename T, int BITS> static hipError_t decode_b(const LowbitDecodeArgs& a, int DP, hipStream_t s) {
  return DP == 32 ? decode_d<T, BITS, 32>(a, s) : DP == 64 ? decode_d<T, BITS, 64>(a, s) : decode_d<T, BITS, 128>(a, s);
}
hipError_t launch_lowbit_decode(const LowbitDecodeArgs& a, bool bf16_in, int bits, int DP, hipStream_t s) {
  if (bf16_in) return bits == 4 ? decode_b<bf16, 4>(a, DP, s) : decode_b<bf16, 8>(a, DP, s);
  return bits == 4 ? decode_b<float, 4>(a, DP, s) : decode_b<float, 8>(a, DP, s);
}

// How a call is cut up.  A workgroup of 4 lb_waves waves has a CU to itself; smaller ones share it.
//  * More workgroups than CUs: of 4 waves, so that one's first loads and last sums pass beside another's work (4 bits, 64 x
//    16 / 16 heads of 2052 slots, d 64, 47.4 us with workgroups of 12 and 38.9 of 4; of 300 slots 25.5, 12.2; 64 x 32 / 8, 8200
//    slots, d 128 104.6, 101.4), unless the cache is long and its last round would leave a fifth of the CUs idle (below).
//  * Else caches of up to four blocks of 32 slots a wave of a large workgroup: one workgroup for all of it, whose one launch
//    is shorter than two.
//  * As many of the large workgroups as CUs, or nearly: no split either (32 x 32 / 8 heads of 4100 slots, d 128 29.2 us, of 4
//    waves 39.0), or as many splits as make that many.
//  * Else splits in workgroups of 4 waves, which fill the CUs in any number (48 x 32 / 8 heads 42.7 us, not split 47.4).
LowbitPlan lowbit_decode_plan(bool bf16_in, int B, int H, int Hk, int d, int S) {
  const int DP = d <= 32 ? 32 : d <= 64 ? 64 : 128, G = H / Hk, gp = bf16_in ? LbHeads<bf16>::GP : LbHeads<float>::GP;
  const int NT = G > gp ? 2 : 1, per = lb_waves(bf16_in ? 2 : 4, DP, NT), big = 4 * per, blocks = (S + 31) / 32;
  LowbitPlan p;
  p.heads = NT * gp;
  const long long wg = (long long)B * Hk * ((G + p.heads - 1) / p.heads), rounds = (wg + CUS - 1) / CUS;
  long long n = 1;
  p.waves = big;
  const bool uneven = wg * 5 < rounds * CUS * 4;
  if (wg > CUS && (blocks <= 4 * big || !uneven)) {
    p.waves = 4;
  } else if (blocks <= 4 * big) {
    p.waves = std::min(big, (blocks + 3) / 4 * 4);
  } else if (uneven) {
    n = CUS / wg;
    if (n * wg * 5 < CUS * 4) {
      p.waves = 4;
      n = std::max(1ll, CUS * per / wg);
    }
    n = std::min<long long>(n, (blocks + p.waves - 1) / p.waves);
  }
  p.chunk = (int)((blocks + n - 1) / n) * 32;
  p.n_split = (S + p.chunk - 1) / p.chunk;
  return p;
}

}  // namespace dfl
