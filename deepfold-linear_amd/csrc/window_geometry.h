// Which pairs of queries and keys the window attention's kernels visit, and where in the table of the relative bias
// their distances lie.  Plain C++ shared by the kernels, the host launch code and a host-side check of the ranges
// (tests/test_window_geometry.py builds it with g++).
#pragma once

#ifndef __HIPCC__
#define __host__
#define __device__
#endif

namespace dfl {

constexpr int REL_MAX_EDGES = 95;   // at most 96 buckets a table
constexpr int REL_MAX_DIST = 2048;  // largest edge

// Bucket of a relative position rel = key - query: mag = |rel| with `both`, else
// max(-rel, 0); bucket = #{k : edge[k] <= mag}, plus n + 1 with `both` and rel > 0.
struct RelSpec {
  int n;     // edges, ascending
  int both;  // both directions: 2 (n + 1) buckets, else n + 1
  int edge[REL_MAX_EDGES];
  __host__ __device__ int buckets() const { return both ? 2 * (n + 1) : n + 1; }
  __host__ __device__ int dist() const { return n ? edge[n - 1] : 0; }  // from here on one bucket a direction
};

__host__ __device__ inline int win_min(int a, int b) { return a < b ? a : b; }
__host__ __device__ inline int win_max(int a, int b) { return a > b ? a : b; }

// Visibility of key j to the query at position t, without the mask.
struct WinVis {
  int off, n_sink, causal;
  unsigned range;
  template <class Args> __host__ __device__ explicit WinVis(const Args& a) {
    const int w = win_min(a.window, a.N);
    off = a.causal ? 0 : w - 1;
    range = (unsigned)(a.causal ? w : 2 * w - 1);
    n_sink = a.n_sink;
    causal = a.causal;
  }
  __host__ __device__ bool near(int t, int j) const { return (unsigned)(t - j + off) < range; }
  __host__ __device__ bool first(int t, int j) const { return (j < n_sink) & ((causal == 0) | (j <= t)); }
  // (combined with & and |: with && and || the 16 elements of a tile become 16 regions of their own execution mask,
  // about 25 instructions each)
  __host__ __device__ bool sees(int t, int j) const { return near(t, j) | first(t, j); }
  // all / none of the pairs of 32 queries from t0 and n keys from j0 on
  __host__ __device__ bool all_near(int t0, int j0, int n = 32) const {
    return near(t0, j0 + n - 1) & near(t0 + 31, j0);
  }
  __host__ __device__ bool none_near(int t0, int j0, int n = 32) const {
    return (t0 + 31 - j0 + off < 0) | (t0 - (j0 + n - 1) + off >= (int)range);
  }
  __host__ __device__ bool none(int t0, int j0, int n = 32) const {
    return none_near(t0, j0, n) & !((j0 < n_sink) & ((causal == 0) | (j0 <= t0 + 31)));
  }
  // whether some of 32 queries from t0 on sees some of 32 keys from j0 on only as a first token
  __host__ __device__ bool some_first(int t0, int j0) const {
    return (j0 < n_sink) & ((causal == 0) | (j0 <= t0 + 31)) & !all_near(t0, j0);
  }
};

// Key tiles of queries t0 .. t1: the first tokens' tiles in front of the band, then the band (and, in both
// directions, the first tokens' tiles behind it).
struct KeyTiles {
  int pre, b0, total;
  template <class Args> __host__ __device__ KeyTiles(const Args& a, int t0, int t1, int BK) {
    const int w = win_min(a.window, a.N);
    const int lo = win_max(0, t0 - w + 1), hi = a.causal ? t1 : win_min(a.N - 1, t1 + w - 1);
    const int nst = (win_min(a.n_sink, a.N) + BK - 1) / BK;
    b0 = lo / BK;
    const int b1 = hi / BK + 1;
    pre = win_min(nst, b0);
    total = pre + (a.causal ? b1 : win_max(b1, nst)) - b0;
  }
  __host__ __device__ int tile(int it) const { return it < pre ? it : b0 + it - pre; }
};

// Tiles of queries that see at most this many keys each (those before row `end`): their D_i is the sum of p dp in a
// pass of its own (window_attn_bwd.hip); of the others, in bf16, the forward keeps what the rounding of o leaves.
constexpr int WIN_EXACT_KEYS = 256;
template <class Args> __host__ __device__ inline bool win_few_keys(const Args& a, int end) {
  const int near = win_min(a.window, a.N), last = a.causal ? win_min(a.M, end) + a.N - a.M : a.N;
  return win_min((a.causal ? near : 2 * near - 1) + win_min(a.n_sink, a.N), last) <= WIN_EXACT_KEYS;
}

// The bias by distance: entry rel_lut_base + t - j of rel_lut_size.  REL_PAD entries more than the table's range on
// both sides hold its end values, so that 32 queries and 32 keys need no clamp where a pair of them is inside the
// range (rel_far() < 0) and, in one direction, one key is not ahead of all the queries (!none, !none_near,
// some_first): the distances of such a pair of tiles reach 62 beyond.
constexpr int REL_PAD = 64;
__host__ __device__ inline int rel_lut_size(const RelSpec& r) {
  return ((r.both ? 2 * r.dist() + 1 : r.dist() + 1) + 2 * REL_PAD + 3) & ~3;
}
__host__ __device__ inline int rel_lut_base(const RelSpec& r) { return (r.both ? r.dist() : 0) + REL_PAD; }
// Where every distance t - j of 32 queries and n keys lies beyond the table's range: the index of its one value, else -1.
__host__ __device__ inline int rel_far(const RelSpec& r, int t0, int j0, int n = 32) {
  const int dist = r.dist();
  if (t0 - (j0 + n - 1) >= dist) return rel_lut_base(r) + dist;
  if (r.both && j0 - (t0 + 31) > dist) return rel_lut_base(r) - dist - 1;
  return -1;
}

}  // namespace dfl
