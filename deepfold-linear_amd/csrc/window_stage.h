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
// the tile in front, written after it.  Rows outside [0, N) or masked, and columns from d on, are zero there (what lies
// in masked rows may be NaN).  A tile inside [0, N) without mask and of full width needs neither clamps nor selects.
template <typename T, int DP, bool FAST> struct RowStage {
  using E = WinEng<T, DP>;
  static constexpr int PER = E::BK * E::NCH / WIN_NT;  // chunks of a thread
  static constexpr int STEP = WIN_NT / E::NCH;         // rows between them
  u32x4 v[PER];
  unsigned ok;  // a bit a chunk: keep it
  __device__ __forceinline__ void load(const T* base, long long stride, int j0, int N, int d, const float* mask) {
    const int r = threadIdx.x / E::NCH, c = threadIdx.x % E::NCH;
    if (FAST && !mask && j0 + E::BK <= N && d == DP) {
      const T* p = base + j0 * stride + (r * stride + c * E::VEC);
#pragma unroll
      for (int n = 0; n < PER; ++n) v[n] = *reinterpret_cast<const u32x4*>(p + n * STEP * stride);
      ok = ~0u;
      return;
    }
    unsigned bits = 0;
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int j = j0 + r + n * STEP, at = min(j, N - 1);
      const T* row = base + at * stride;
      if (FAST) {  // a chunk behind the row's end reads the row's first one
        v[n] = *reinterpret_cast<const u32x4*>(row + (c * E::VEC < d ? c * E::VEC : 0));
        bits |= (unsigned)((j < N) & (c * E::VEC < d)) << n;
      } else {
        v[n] = E::template load<false>(row, c, d);
        bits |= (unsigned)(j < N) << n;
      }
    }
    if (mask) {
#pragma unroll
      for (int n = 0; n < PER; ++n) bits &= ~((unsigned)(mask[min(j0 + r + n * STEP, N - 1)] == 0.f) << n);
    }
    ok = bits;
  }
  __device__ __forceinline__ void store(T* tile) {
    const int r = threadIdx.x / E::NCH, c = threadIdx.x % E::NCH;
    if (__any(ok != ~0u)) {
      const u32x4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int n = 0; n < PER; ++n) v[n] = (ok >> n) & 1u ? v[n] : zero;
    }
#pragma unroll
    for (int n = 0; n < PER; ++n) *E::chunk(tile, r + n * STEP, c) = v[n];
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
    if (mask || j0 + E::BK > N) {
      const int lane = threadIdx.x & 63, j = j0 + lane;
      const bool in = (lane < E::BK) & (j < N);
      bits = __ballot(in && (!mask || mask[in ? j : 0] != 0.f));
    } else {
      bits = ~0ull;
    }
  }
  __device__ __forceinline__ void store(T* sk, T* sv, unsigned* smask) {
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
