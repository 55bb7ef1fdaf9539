// One token's attention over a rolling cache in 8 or 4 bits.
//
// Codes become bf16 operands of 16x16x32 matrix instructions in registers, exactly (a code has at most 7 bits, its scale
// is a power of two), straight from the loads: no LDS between.  In vector instructions alone the products of four heads
// would take longer than the codes take to arrive.  A wave takes 32 slots at a time:
//   scores (slots x heads): A = 16 rows of keys, lane l the row l % 16 and a quarter l / 16 of its elements, as they
//     lie in memory; B = the queries with the same elements.  Accumulator: lane = head l % 16, slots 4 (l / 16) + r.
//   outputs (heads x columns): A = the weights, head l % 16, slots 4 (l / 16) + r of both halves: they stay in their lane;
//     B = 16 columns of the values of these slots: lane l loads the elements l % 16 * DP / 16 .. of each of its slots.
// The 16 rows of the weights hold GP heads in TERMS parts: bf16 results take two bf16 numbers for a weight (16 bits of
// it), fp32 results three (24 bits), so no weight is rounded to 8 bits and the matrix rows would be idle otherwise.  fp32
// queries are three bf16 numbers, products of their own.  Sums, references and outputs are fp32.
#include "lowbit_args.h"
#include "lowbit_codes.h"
#include "window_engine.h"

#include <initializer_list>

namespace dfl {

template <typename T> struct LbHeads {
  static constexpr int TERMS = sizeof(T) == 2 ? 2 : 4;  // parts of a weight (the fourth of fp32 is zero)
  static constexpr int GP = 16 / TERMS;                 // heads of a tile
  static constexpr int QT = sizeof(T) == 2 ? 1 : 3;     // parts of a query
};
// A reference is moved when a score passes it by more than this: weights stay below 2^8.
constexpr float LB_LAZY = 8.f;

__device__ __forceinline__ int lb_position(int s, int last, int n_sink, int window) {
  return s < n_sink ? s : s + (last - s) / window * window;
}
__device__ __forceinline__ unsigned bf16_pair(float lo, float hi) {  // upper halves: exact where the values have 8 bits
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

union LbFrag {
  unsigned u[4];
  bf16x8 v;
};

template <typename T, int BITS, int DP, int NT, bool REL>
__global__ void __launch_bounds__(256) lowbit_decode_kernel(LowbitDecodeArgs a) {
  using Hd = LbHeads<T>;
  constexpr int GP = Hd::GP, QT = Hd::QT, GB = NT * GP;
  constexpr int KF = DP / 32;            // matrix instructions of a score tile; fragments of a lane's quarter row
  constexpr int KW = DP * BITS / 128;    // dwords of a lane's quarter row: KF of 4 bits, 2 KF of 8
  constexpr int NC = DP / 16;            // columns of a lane
  constexpr int VB = NC * BITS / 8;      // bytes of them: 1, 2, 4 or 2, 4, 8
  constexpr int VW = (VB + 3) / 4;
  extern __shared__ __align__(16) unsigned char smem[];
  float* s_ml = reinterpret_cast<float*>(smem);  // [4][GB][2]
  float* s_o = s_ml + 4 * GB * 2;                // [4][GB][DP]
  uint8_t* s_own = reinterpret_cast<uint8_t*>(s_o + 4 * GB * DP);  // [2][DP * BITS / 8] the token's own codes
  uint8_t* s_exp = s_own + 2 * DP * BITS / 8;                      // [2][4]
  float* s_tab = reinterpret_cast<float*>(s_exp + 8);              // [GB][buckets]
  uint8_t* s_lut = reinterpret_cast<uint8_t*>(s_tab + (REL ? GB * a.rel.buckets() : 0));
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, h = lane >> 4;
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

  // The token's own codes: from the call's rows into LDS, and into the cache by one workgroup.
  if (mine && wave < 2 && lane < nch) {
    const T* row = wave ? reinterpret_cast<const T*>(a.v) + b * a.vsb + hk * a.vsh
                        : reinterpret_cast<const T*>(a.k) + b * a.ksb + hk * a.ksh;
    float e[8];
    unsigned w[BITS / 4];
    load8<T, false>(row, lane, a.d, e);
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
    for (int e = threadIdx.x; e < gn * nb; e += 256) s_tab[e] = a.table[(size_t)h0 * nb + e] * LOG2E;
    for (int e = threadIdx.x; e <= dist; e += 256) s_lut[e] = (uint8_t)rel_bucket(a.rel, -e);
  }
  // The queries: lane's column n is head n % GP of a tile, elements DP / 4 * h .. of it.  They take the scale's power of
  // two, which changes none of their digits; the scores take the rest of it, a factor from 1 to 2.
  const float sc0 = a.scale * LOG2E, two = __uint_as_float(__float_as_uint(sc0) & 0x7f800000u), sc = sc0 / two;
  LbFrag q[NT][QT][KF];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int g = i * GP + n % GP;
    const T* row = reinterpret_cast<const T*>(a.q) + b * a.qsb + (h0 + min(g, gn - 1)) * a.qsh;
#pragma unroll
    for (int f = 0; f < KF; ++f)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = DP / 4 * h + 8 * f + e;
        float rest = g < gn && at < a.d ? to_f32(row[at]) * two : 0.f;
#pragma unroll
        for (int p = 0; p < QT; ++p) {
          // parts cut off, not rounded: a finite query has no infinite part
          const bool fine = fabsf(rest) < INFINITY;
          const float part = fine ? __uint_as_float(__float_as_uint(rest) & 0xffff0000u) : rest;
          q[i][p][f].v[e] = (bf16)part;
          rest = fine ? rest - part : 0.f;
        }
      }
  }
  __syncthreads();

  const int term = n / GP;
  const float sel1 = term >= 1 ? -1.f : 0.f, sel2 = term >= 2 ? -1.f : 0.f;
  const int kg = DP / 4 * h / 32, vg = n * NC / 32;   // groups of the lane's key and value elements
  const bool kin = kg < groups, vin = vg < groups;    // (96 of 128 elements: the last quarter has none)
  const int kge = min(kg, groups - 1), vge = min(vg, groups - 1);
  f32x4 o[NT][NC];
  float m[NT], l[NT];
  unsigned bad = 0;
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    m[i] = NEG_BIG, l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) o[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  struct Raw {
    unsigned k[2][KW], v[8][VW];
    unsigned ke[2], ve[2];
  };
  const int kofs = h * (KW * 4), vofs = n * VB;
  auto load = [&](Raw& r, int s0) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int s = min(s0 + 16 * u + n, end - 1);
      const unsigned* at = reinterpret_cast<const unsigned*>(kc + s * a.kc.sn + (kin ? kofs : 0));
#pragma unroll
      for (int i = 0; i < KW; ++i) r.k[u][i] = at[i];
      r.ke[u] = ke[kge * a.kc.esg + s];
      // four slots' bytes; the last dword of a group where these would lie behind it (they are masked then)
      const int s4 = min(s0 + 16 * u + 4 * h, (S - 1) & ~3);
      r.ve[u] = *reinterpret_cast<const unsigned*>(ve + vge * a.vc.esg + s4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int sv = min(s0 + 16 * u + 4 * h + j, end - 1);
        const uint8_t* p = vc + sv * a.vc.sn + (vin ? vofs : 0);
        if constexpr (VB == 1) r.v[4 * u + j][0] = *p;
        else if constexpr (VB == 2) r.v[4 * u + j][0] = *reinterpret_cast<const unsigned short*>(p);
        else
#pragma unroll
          for (int i = 0; i < VW; ++i) r.v[4 * u + j][i] = reinterpret_cast<const unsigned*>(p)[i];
      }
    }
  };
  auto step = [&](Raw& r, int s0) {
    if (mine && s0 <= own && own < s0 + 32) {  // the token's own slot, as its codes stand
      const int at = own - s0;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (16 * u + n == at) {
          const unsigned* p = reinterpret_cast<const unsigned*>(s_own + (kin ? kofs : 0));
#pragma unroll
          for (int i = 0; i < KW; ++i) r.k[u][i] = p[i];
          r.ke[u] = s_exp[kge];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (16 * u + 4 * h + j == at) {
            const uint8_t* p = s_own + DP * BITS / 8 + (vin ? vofs : 0);
            if constexpr (VB == 1) r.v[4 * u + j][0] = *p;
            else if constexpr (VB == 2) r.v[4 * u + j][0] = *reinterpret_cast<const unsigned short*>(p);
            else
#pragma unroll
              for (int i = 0; i < VW; ++i) r.v[4 * u + j][i] = reinterpret_cast<const unsigned*>(p)[i];
            r.ve[u] = (r.ve[u] & ~(255u << (8 * j))) | (unsigned)s_exp[4 + vge] << (8 * j);
          }
      }
    }
    const bool whole = s0 + 32 <= end;
    if (!whole) {  // slots that are not in use: their exponents are not looked at
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (s0 + 16 * u + n >= end) r.ke[u] = 0;
        const int left = end - (s0 + 16 * u + 4 * h);
        if (left < 4) r.ve[u] = left <= 0 ? 0u : r.ve[u] & ((1u << (8 * left)) - 1);
      }
    }
    // scores
    f32x4 y[2][NT];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float ks = kin ? lb_scale(r.ke[u]) : 0.f;
      bad |= kin ? (r.ke[u] + 1) & 256u : 0u;
#pragma unroll
      for (int i = 0; i < NT; ++i) y[u][i] = f32x4{0.f, 0.f, 0.f, 0.f};
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
    // weights
    LbFrag w[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      float mx = NEG_BIG;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int s = s0 + 16 * u + 4 * h + j;
          float v = y[u][i][j] * sc;
          if (REL) {
            const int bk = s_lut[min(t - lb_position(min(s, end - 1), t, a.n_sink, a.window), a.rel.dist())];
            v += s_tab[min(i * GP + n % GP, gn - 1) * a.rel.buckets() + bk];
          }
          if (!whole) v = s < end ? v : -INFINITY;
          y[u][i][j] = v;
          mx = fmaxf(mx, v);
        }
      if (__any(mx > m[i] + LB_LAZY)) {
        mx = max_groups(fmaxf(mx, m[i]));
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
      const unsigned e = vin ? r.ve[u] : 0u;
      bad |= (((e & 0x7f7f7f7fu) + 0x01010101u) & e) & 0x80808080u;
#pragma unroll
      for (int j = 0; j < 4; ++j) vs[4 * u + j] = lb_scale((e >> (8 * j)) & 255u);
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
  {
    int s0 = begin + 32 * wave;
    if (s0 < end) {
      Raw now, next;
      load(now, s0);
      for (; s0 + 128 < end; s0 += 128) {
        load(next, s0 + 128);
        step(now, s0);
        now = next;
      }
      step(now, s0);
    }
  }

  // The waves' parts: weights' parts and lanes joined, then the waves in LDS.
  const bool poison = __any(bad != 0);
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
  for (int e = threadIdx.x; e < gn * DP; e += 256) {
    const int g = e / DP, col = e % DP;
    float mx = NEG_BIG;
#pragma unroll
    for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s_ml[(r * GB + g) * 2]);
    float sl = 0.f, so = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float al = fast_exp2(s_ml[(r * GB + g) * 2] - mx);
      sl = __builtin_fmaf(s_ml[(r * GB + g) * 2 + 1], al, sl);
      so = __builtin_fmaf(s_o[(r * GB + g) * DP + col], al, so);
    }
    const size_t head = (size_t)b * a.H + h0 + g;
    if (a.n_split == 1) {
      if (col < a.d) reinterpret_cast<T*>(a.o)[head * a.d + col] = from_f32<T>(sl == 0.f ? 0.f : so / sl);
    } else {
      float* part = a.part + (head * a.n_split + sp) * (DP + 2);
      if (col == 0) part[0] = mx, part[1] = sl;
      part[2 + col] = so;
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
  const size_t lds = (size_t)4 * GB * (DP + 2) * 4 + 2 * DP * BITS / 8 + 8 +
                     (REL ? (size_t)GB * a.rel.buckets() * 4 + a.rel.dist() + 1 : 0);
  auto kern = lowbit_decode_kernel<T, BITS, DP, NT, REL>;
  hipError_t e = set_lds_limit((const void*)kern, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3((unsigned)(a.B * a.Hk * nhg * a.n_split)), dim3(256), lds, s, a);
  if ((e = hipGetLastError()) != hipSuccess || a.n_split == 1) return e;
  hipLaunchKernelGGL((lowbit_join_kernel<T, DP>), dim3((unsigned)(a.B * a.H)), dim3(128), a.n_split * 4, s, a);
  return hipGetLastError();
}
template <typename T, int BITS, int DP> static hipError_t decode_d(const LowbitDecodeArgs& a, hipStream_t s) {
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
int lowbit_decode_heads(bool bf16_in, int G) {
  const int gp = bf16_in ? LbHeads<bf16>::GP : LbHeads<float>::GP;
  return G > gp ? 2 * gp : gp;
}

}  // namespace dfl
