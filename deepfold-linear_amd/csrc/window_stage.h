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

// Stages rows j0 .. j0 + BK - 1 of one operand; rows outside [0, N) or masked are zero (their values may be NaN).
template <typename T, int DP, bool FAST>
__device__ __forceinline__ void stage_rows(T* tile, const T* base, long long stride, int j0, int N, int d,
                                           const float* mask) {
  using E = WinEng<T, DP>;
  for (int e = threadIdx.x; e < E::BK * E::NCH; e += WIN_NT) {
    const int r = e / E::NCH, c = e % E::NCH, j = j0 + r;
    const bool ok = j >= 0 && j < N && (!mask || mask[j] != 0.f);
    *E::chunk(tile, r, c) = E::template load<FAST>(ok ? base + (size_t)j * stride : nullptr, c, d);
  }
}

// One key tile: K, V and the bits of its keys that are inside and unmasked.
template <typename T, int DP, bool FAST>
__device__ __forceinline__ void stage_tile(T* sk, const T* kb, long long ksn, T* sv, const T* vb, long long vsn,
                                           unsigned* smask, int j0, int N, int d, const float* mask) {
  using E = WinEng<T, DP>;
  stage_rows<T, DP, FAST>(sk, kb, ksn, j0, N, d, mask);
  stage_rows<T, DP, FAST>(sv, vb, vsn, j0, N, d, mask);
  if (threadIdx.x < 64) {
    const int j = j0 + threadIdx.x;
    const bool in = (int)threadIdx.x < E::BK && j < N;
    const uint64_t ok = __ballot(in && (!mask || mask[in ? j : 0] != 0.f));
    if (threadIdx.x == 0) {
      smask[0] = (unsigned)ok;
      smask[1] = (unsigned)(ok >> 32);
    }
  }
}

}  // namespace dfl
