// Which key tiles a workgroup of the window attention visits, and their staging into LDS.
#pragma once
#include "window_engine.h"

namespace dfl {

// Key tiles of queries t0 .. t1: the first tokens' tiles in front of the band, then the band (and, in both
// directions, the first tokens' tiles behind it).
struct KeyTiles {
  int pre, b0, total;
  __device__ __forceinline__ KeyTiles(const WinArgs& a, int t0, int t1, int BK) {
    const int w = min(a.window, a.N);
    const int lo = max(0, t0 - w + 1), hi = a.causal ? t1 : min(a.N - 1, t1 + w - 1);
    const int nst = (min(a.n_sink, a.N) + BK - 1) / BK;
    b0 = lo / BK;
    const int b1 = hi / BK + 1;
    pre = min(nst, b0);
    total = pre + (a.causal ? b1 : max(b1, nst)) - b0;
  }
  __device__ __forceinline__ int tile(int it) const { return it < pre ? it : b0 + it - pre; }
};

// Rows j0 .. j0 + BK - 1 of one operand on their way to LDS: issued as loads into registers before the product of
// the tile in front, written after it.  Rows outside [0, N) or masked are zero there (their values may be NaN).
template <typename T, int DP, bool FAST> struct RowStage {
  using E = WinEng<T, DP>;
  static constexpr int PER = E::BK * E::NCH / WIN_NT;  // chunks of a thread
  u32x4 v[PER];
  unsigned ok;  // a bit a chunk
  __device__ __forceinline__ void load(const T* base, long long stride, int j0, int N, int d, const float* mask) {
    ok = 0;
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int e = threadIdx.x + n * WIN_NT, r = e / E::NCH, j = j0 + r, at = min(j, N - 1);
      v[n] = E::template load<FAST>(base + (size_t)at * stride, e % E::NCH, d);
      ok |= (unsigned)((j < N) & (!mask || mask[at] != 0.f)) << n;
    }
  }
  __device__ __forceinline__ void store(T* tile) const {
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int e = threadIdx.x + n * WIN_NT;
      const u32x4 zero = {0u, 0u, 0u, 0u};
      *E::chunk(tile, e / E::NCH, e % E::NCH) = (ok >> n) & 1u ? v[n] : zero;
    }
  }
};

// One key tile: K, V and the bits of its keys that are inside and unmasked (the first wave's).
template <typename T, int DP, bool FAST> struct KeyStage {
  using E = WinEng<T, DP>;
  RowStage<T, DP, FAST> k, v;
  uint64_t bits;
  __device__ __forceinline__ void load(const T* kb, long long ksn, const T* vb, long long vsn, int j0, int N, int d,
                                       const float* mask) {
    k.load(kb, ksn, j0, N, d, mask);
    v.load(vb, vsn, j0, N, d, mask);
    if (threadIdx.x < 64) {
      const int j = j0 + threadIdx.x;
      const bool in = ((int)threadIdx.x < E::BK) & (j < N);
      bits = __ballot(in && (!mask || mask[in ? j : 0] != 0.f));
    }
  }
  __device__ __forceinline__ void store(T* sk, T* sv, unsigned* smask) const {
    k.store(sk);
    v.store(sv);
    if (threadIdx.x == 0) {
      smask[0] = (unsigned)bits;
      smask[1] = (unsigned)(bits >> 32);
    }
  }
};

// Four consecutive columns c .. c + 3 of a result row of d columns.
template <typename T, bool FAST> __device__ __forceinline__ void store4(T* row, int c, int d, f32x4 x) {
  typedef __attribute__((__vector_size__(4 * sizeof(T)))) T vec;
  if (FAST) {
    if (c < d) {
      vec o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = from_f32<T>(x[e]);
      *reinterpret_cast<vec*>(row + c) = o;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < d) row[c + e] = from_f32<T>(x[e]);
  }
}

}  // namespace dfl
