// The rolling cache of the window attention: copy of a prompt into it, and one token's attention over it.
//
// Position p < n_sink lies in slot p, any other in slot n_sink + (p - n_sink) % window: what the slots hold once
// token t is in is exactly what t sees, so a token reads each slot in use once and nothing else.
//
// Bounds: the cache's bytes, once for four query heads of a key head (each group of heads more reads them once more: 8
// sequences of 4100 slots, 32 / 4 heads, d 128, bf16, 67 MB: 38 us).  32 sequences of 4100 slots, 32 / 8 heads, d 128,
// bf16, 537 MB: 106 us, 5.0 TB/s of the 6.2-6.4 that a copy or read reaches (join 5 us more); 270 MB of prompts into 32
// caches: 43 us, 6.2 TB/s.  One sequence of 1028 slots, 16 / 4 heads, d 64: 7 + 3.6 us, both of them latency.
#include "window_engine.h"

#include <algorithm>

namespace dfl {

// Latest position <= last that slot s holds, -1 if none.
__device__ __forceinline__ int slot_position(int s, int last, int n_sink, int window) {
  if (s > last) return -1;
  return s < n_sink ? s : s + (last - s) / window * window;
}

template <typename T, bool FAST> __global__ void __launch_bounds__(256) cache_fill_kernel(CacheFillArgs a) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int nch = (a.d + VEC - 1) / VEC, S = a.n_sink + a.window;
  const int bh = blockIdx.y, b = bh / a.Hk, hk = bh % a.Hk;
  const int last = max(min(a.lengths[b], a.N), 0) - 1;  // (a length of -2^31 has no predecessor)
  const long long e = (long long)blockIdx.x * 256 + threadIdx.x;  // (slot, chunk)
  const int s = (int)(e / nch), c = (int)(e % nch);
  if (s >= S) return;
  const int p = slot_position(s, last, a.n_sink, a.window);
  if (p < 0) return;
  const T* k = reinterpret_cast<const T*>(a.k) + b * a.ksb + hk * a.ksh + (size_t)p * a.ksn + c * VEC;
  const T* v = reinterpret_cast<const T*>(a.v) + b * a.vsb + hk * a.vsh + (size_t)p * a.vsn + c * VEC;
  T* ko = reinterpret_cast<T*>(a.kc) + b * a.kcsb + hk * a.kcsh + (size_t)s * a.kcsn + c * VEC;
  T* vo = reinterpret_cast<T*>(a.vc) + b * a.vcsb + hk * a.vcsh + (size_t)s * a.vcsn + c * VEC;
  if (FAST) {
    *reinterpret_cast<u32x4*>(ko) = *reinterpret_cast<const u32x4*>(k);
    *reinterpret_cast<u32x4*>(vo) = *reinterpret_cast<const u32x4*>(v);
  } else {
    for (int i = 0; i < VEC && c * VEC + i < a.d; ++i) ko[i] = k[i], vo[i] = v[i];
  }
}

// x summed over the L lanes (a power of two, aligned) that share a row
template <int L> __device__ __forceinline__ float row_sum(float x) {
  if (L >= 2) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xb1, 0xf, 0xf, false));
  if (L >= 4) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4e, 0xf, 0xf, false));
  if (L >= 8) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x141, 0xf, 0xf, false));
  if (L >= 16) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x140, 0xf, 0xf, false));
  if (L >= 32) x = xor16_pair(x, false);
  return x;
}

constexpr int DEC_U = 4;

// One (sample, key head, group of up to GB query heads, split of the slots) a workgroup.  L lanes hold a row, 16
// bytes each; a wave takes 64 / L rows at a time, each lane group with a running reference, sum and output of its
// own, joined in LDS at the end.
template <typename T, int DP, int GB, bool FAST, bool REL>
__global__ void __launch_bounds__(256) window_decode_kernel(DecodeArgs a) {
  using E = WinEng<T, DP>;
  constexpr int VEC = E::VEC, L = E::NCH, RPW = 64 / L, NG = 4 * RPW;  // row groups of the workgroup
  extern __shared__ __align__(16) unsigned char smem[];
  float* s_ml = reinterpret_cast<float*>(smem);  // [NG][GB][2]
  float* s_o = s_ml + NG * GB * 2;               // [NG][GB][DP]
  float* s_tab = s_o + NG * GB * DP;             // [GB][buckets]
  uint8_t* s_lut = reinterpret_cast<uint8_t*>(s_tab + (REL ? GB * a.rel.buckets() : 0));
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane % L, rg = wave * RPW + lane / L;
  const int G = a.H / a.Hk, nhg = (G + GB - 1) / GB;
  int x = blockIdx.x;
  const int sp = x % a.n_split;
  x /= a.n_split;
  const int hg = x % nhg, bh = x / nhg, b = bh / a.Hk, hk = bh % a.Hk;
  const int g0 = hg * GB, gn = min(GB, G - g0), h0 = hk * G + g0;
  const int t = a.lengths[b], S = a.n_sink + a.window;
  const int used = t < 0 ? 0 : (t >= S ? S : t + 1);
  const int own = t < a.n_sink ? t : a.n_sink + (t - a.n_sink) % a.window;  // the token's own slot
  if (REL) {
    const int nb = a.rel.buckets(), dist = a.rel.dist();
    for (int e = threadIdx.x; e < gn * nb; e += 256) s_tab[e] = a.table[(size_t)h0 * nb + e] * LOG2E;
    for (int e = threadIdx.x; e <= dist; e += 256) s_lut[e] = (uint8_t)rel_bucket(a.rel, -e);
    __syncthreads();
  }
  const float sc = a.scale * LOG2E;
  float q[GB][VEC], o[GB][VEC], m[GB], l[GB];
#pragma unroll
  for (int g = 0; g < GB; ++g) {
    const T* row = g < gn ? reinterpret_cast<const T*>(a.q) + b * a.qsb + (h0 + g) * a.qsh : nullptr;
    const u32x4 w = E::template load<FAST>(row, c, a.d);
    T e[VEC];
    __builtin_memcpy(e, &w, 16);
#pragma unroll
    for (int i = 0; i < VEC; ++i) q[g][i] = to_f32(e[i]) * sc, o[g][i] = 0.f;
    m[g] = NEG_BIG;
    l[g] = 0.f;
  }
  T* kc = reinterpret_cast<T*>(a.kc) + b * a.kcsb + hk * a.kcsh;
  T* vc = reinterpret_cast<T*>(a.vc) + b * a.vcsb + hk * a.vcsh;
  const T* kn = reinterpret_cast<const T*>(a.k) + b * a.ksb + hk * a.ksh;
  const T* vn = reinterpret_cast<const T*>(a.v) + b * a.vsb + hk * a.vsh;
  const int s1 = min(used, (sp + 1) * a.chunk);
  // DEC_U rows of a lane group at a time: their loads in flight together, one move of the reference for all
  for (int s0 = sp * a.chunk + rg; s0 < s1; s0 += NG * DEC_U) {
    u32x4 kw[DEC_U], vw[DEC_U];
#pragma unroll
    for (int u = 0; u < DEC_U; ++u) {
      const int s = min(s0 + u * NG, s1 - 1);
      const bool mine = s == own;
      kw[u] = E::template load<FAST>(mine ? kn : kc + (size_t)s * a.kcsn, c, a.d);
      vw[u] = E::template load<FAST>(mine ? vn : vc + (size_t)s * a.vcsn, c, a.d);
    }
    float y[DEC_U][GB];
#pragma unroll
    for (int u = 0; u < DEC_U; ++u) {
      const int s = s0 + u * NG;
      T ke[VEC];
      __builtin_memcpy(ke, &kw[u], 16);
      int bk = 0;
      if (REL) bk = s_lut[min(t - slot_position(min(s, s1 - 1), t, a.n_sink, a.window), a.rel.dist())];
#pragma unroll
      for (int g = 0; g < GB; ++g) {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) x = __builtin_fmaf(q[g][i], to_f32(ke[i]), x);
        x = row_sum<L>(x);
        if (REL) x += s_tab[min(g, gn - 1) * a.rel.buckets() + bk];
        y[u][g] = s < s1 ? x : -INFINITY;
      }
      if (s == own && s < s1 && hg == 0) {  // the token enters the cache; no workgroup reads its slot
        T ve[VEC];
        __builtin_memcpy(ve, &vw[u], 16);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (c * VEC + i < a.d) {
            kc[(size_t)s * a.kcsn + c * VEC + i] = ke[i];
            vc[(size_t)s * a.vcsn + c * VEC + i] = ve[i];
          }
      }
    }
#pragma unroll
    for (int g = 0; g < GB; ++g) {
      float mx = m[g];
#pragma unroll
      for (int u = 0; u < DEC_U; ++u) mx = fmaxf(mx, y[u][g]);
      const float al = fast_exp2(m[g] - mx);
      m[g] = mx;
      l[g] *= al;
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[g][i] *= al;
    }
#pragma unroll
    for (int u = 0; u < DEC_U; ++u) {
      T ve[VEC];
      __builtin_memcpy(ve, &vw[u], 16);
#pragma unroll
      for (int g = 0; g < GB; ++g) {
        const float p = fast_exp2(y[u][g] - m[g]);
        l[g] += p;
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[g][i] = __builtin_fmaf(p, to_f32(ve[i]), o[g][i]);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < GB; ++g) {
    if (c == 0) {
      s_ml[(rg * GB + g) * 2] = m[g];
      s_ml[(rg * GB + g) * 2 + 1] = l[g];
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) s_o[(rg * GB + g) * DP + c * VEC + i] = o[g][i];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < gn * DP; e += 256) {
    const int g = e / DP, col = e % DP;
    float mx = NEG_BIG;
    for (int r = 0; r < NG; ++r) mx = fmaxf(mx, s_ml[(r * GB + g) * 2]);
    float sl = 0.f, so = 0.f;
    for (int r = 0; r < NG; ++r) {
      const float al = fast_exp2(s_ml[(r * GB + g) * 2] - mx);
      sl = __builtin_fmaf(s_ml[(r * GB + g) * 2 + 1], al, sl);
      so = __builtin_fmaf(s_o[(r * GB + g) * DP + col], al, so);
    }
    const size_t head = (size_t)b * a.H + h0 + g;
    if (a.n_split == 1) {
      if (col < a.d) reinterpret_cast<T*>(a.o)[head * a.d + col] = from_f32<T>(sl > 0.f ? so / sl : 0.f);
    } else {
      float* part = a.part + (head * a.n_split + sp) * (DP + 2);
      if (col == 0) part[0] = mx, part[1] = sl;
      part[2 + col] = so;
    }
  }
}

// The splits' outputs joined, in split order: a workgroup a head, a wave or more, the splits' references and sums in
// LDS first so that the loop over the outputs has only independent loads.
template <typename T, int DP> __global__ void __launch_bounds__(128) window_decode_join_kernel(DecodeArgs a) {
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
  reinterpret_cast<T*>(a.o)[head * a.d + col] = from_f32<T>(l > 0.f ? o / l : 0.f);
}

template <typename T> static bool aligned(const void* p, std::initializer_list<long long> strides) {
  bool ok = ((uintptr_t)p & 15u) == 0;
  for (long long s : strides) ok = ok && ((s * (long long)sizeof(T)) & 15) == 0;
  return ok;
}

template <typename T> static hipError_t fill_t(const CacheFillArgs& a, hipStream_t s) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const bool fast = a.d % VEC == 0 && aligned<T>(a.k, {a.ksb, a.ksh, a.ksn}) && aligned<T>(a.v, {a.vsb, a.vsh, a.vsn}) &&
                    aligned<T>(a.kc, {a.kcsb, a.kcsh, a.kcsn}) && aligned<T>(a.vc, {a.vcsb, a.vcsh, a.vcsn});
  const long long per = (long long)(a.n_sink + a.window) * ((a.d + VEC - 1) / VEC);
  const dim3 grid((unsigned)((per + 255) / 256), a.B * a.Hk);
  if (fast) hipLaunchKernelGGL((cache_fill_kernel<T, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((cache_fill_kernel<T, false>), grid, dim3(256), 0, s, a);
  return hipGetLastError();
}
hipError_t launch_cache_fill(const CacheFillArgs& a, bool bf16_in, hipStream_t s) {
  return bf16_in ? fill_t<bf16>(a, s) : fill_t<float>(a, s);
}

template <typename T, int DP, int GB, bool FAST, bool REL> static hipError_t decode_l(const DecodeArgs& a, hipStream_t s) {
  using E = WinEng<T, DP>;
  constexpr int NG = 4 * (64 / E::NCH);
  const int G = a.H / a.Hk, nhg = (G + GB - 1) / GB;
  const size_t lds = (size_t)NG * GB * (DP + 2) * 4 + (REL ? (size_t)GB * a.rel.buckets() * 4 + a.rel.dist() + 1 : 0);
  auto kern = window_decode_kernel<T, DP, GB, FAST, REL>;
  hipError_t e = set_lds_limit((const void*)kern, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3((unsigned)(a.B * a.Hk * nhg * a.n_split)), dim3(256), lds, s, a);
  if ((e = hipGetLastError()) != hipSuccess || a.n_split == 1) return e;
  hipLaunchKernelGGL((window_decode_join_kernel<T, DP>), dim3((unsigned)(a.B * a.H)), dim3(128), a.n_split * 4, s, a);
  return hipGetLastError();
}
template <typename T, int DP, int GB> static hipError_t decode_g(const DecodeArgs& a, bool fast, hipStream_t s) {
  if (a.table) return fast ? decode_l<T, DP, GB, true, true>(a, s) : decode_l<T, DP, GB, false, true>(a, s);
  return fast ? decode_l<T, DP, GB, true, false>(a, s) : decode_l<T, DP, GB, false, false>(a, s);
}
template <typename T, int DP> static hipError_t decode_d(const DecodeArgs& a, hipStream_t s) {
  const bool fast = a.d % WinEng<T, DP>::VEC == 0 && aligned<T>(a.q, {a.qsb, a.qsh}) && aligned<T>(a.k, {a.ksb, a.ksh}) &&
                    aligned<T>(a.v, {a.vsb, a.vsh}) && aligned<T>(a.kc, {a.kcsb, a.kcsh, a.kcsn}) &&
                    aligned<T>(a.vc, {a.vcsb, a.vcsh, a.vcsn});
  const int G = a.H / a.Hk;
  return G == 1 ? decode_g<T, DP, 1>(a, fast, s) : G == 2 ? decode_g<T, DP, 2>(a, fast, s) : decode_g<T, DP, 4>(a, fast, s);
}
hipError_t launch_window_decode(const DecodeArgs& a, bool bf16_in, int DP, hipStream_t s) {
  if (bf16_in)
    return DP == 32 ? decode_d<bf16, 32>(a, s) : DP == 64 ? decode_d<bf16, 64>(a, s) : decode_d<bf16, 128>(a, s);
  return DP == 32 ? decode_d<float, 32>(a, s) : DP == 64 ? decode_d<float, 64>(a, s) : decode_d<float, 128>(a, s);
}

}  // namespace dfl
