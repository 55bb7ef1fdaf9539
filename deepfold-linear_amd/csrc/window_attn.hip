// Attention over a sliding window and a few first tokens, forward.
//
// Query i stands at position t = i + N - M; it sees the keys t - window < j <= t (both
// directions: |t - j| < window) and the keys j < n_sink (causal: j <= t).
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp2(y_ij - m_i),
//   y_ij = log2(e) (scale q_i.k_j + table[bucket(j - t)])
// A workgroup owns 128 queries of one head, a wave 32 of them; the keys it can see stream through LDS once, in tiles of
// 64, with the running reference m_i and the sum in registers.  The next tile's loads go straight into the other LDS
// buffer during this one's products.
//
// Bounds (MI355X, bf16, d 128, window 2048, 32 / 8 heads of 8192 tokens with a table, 240 GFLOP): 322 us among other
// passes, 745 TFLOP/s (379 us under a kernel trace), against 190 us at the rate of a large library product and 115 us at
// what the matrix instructions alone reach.
// A wave's step of 64 keys is 32 matrix instructions (1024 cycles of its SIMD) and about 220 others (1100 cycles with
// the 32 exponentials at a quarter rate); two waves a SIMD overlap the two in part, the rest is their barrier and LDS
// latency.  32 queries a wave and not 64: twice the queries would halve the LDS reads, which take 22 % of the time, but
// leave one wave a SIMD and nothing to cover the exponentials.
#include "window_engine.h"
#include "window_stage.h"

namespace dfl {

// A row's reference moves only when a score exceeds it by this much (log2): the weights stay below 2^8, the output
// rows are rescaled once or twice a row instead of once a tile.
constexpr float WIN_SLACK = 8.f;

template <typename T, int DP, bool FAST, bool REL>
__global__ void __launch_bounds__(WIN_NT, sizeof(T) == 4 && DP == 128 ? 1 : 2) window_fwd_kernel(WinArgs a) {
  using E = WinEng<T, DP>;
  extern __shared__ __align__(16) unsigned char smem[];
  T* sk = reinterpret_cast<T*>(smem);  // [2] key tiles, [2] value tiles
  T* sv = sk + 2 * E::TILE;
  float* lut = reinterpret_cast<float*>(sv + 2 * E::TILE);
  int* edge = reinterpret_cast<int*>(lut + (REL ? rel_lut_size(a.rel) : 0));
  const int lane = threadIdx.x & 63, h32 = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // uniform: tile tests are scalar

  const int G = a.H / a.Hk, nqt = (a.M + WIN_RES - 1) / WIN_RES;
  int x = xcd_order(blockIdx.x, gridDim.x);
  const int g = x % G;
  x /= G;
  const int qt = x % nqt, bhk = x / nqt, b = bhk / a.Hk, hk = bhk % a.Hk, h = hk * G + g;
  const int shift = a.N - a.M;  // position of query 0
  const T* kb = reinterpret_cast<const T*>(a.k) + b * a.ksb + hk * a.ksh;
  const T* vb = reinterpret_cast<const T*>(a.v) + b * a.vsb + hk * a.vsh;
  const float* mask = a.mask ? a.mask + (size_t)b * a.N : nullptr;
  const WinVis vis(a);

  const KeyTiles kt(a, qt * WIN_RES + shift, min(a.M, (qt + 1) * WIN_RES) - 1 + shift, E::BK);
  const RowLoader<T, DP, FAST> lk(a.ksn, a.N, a.d), lv(a.vsn, a.N, a.d);
  lk.issue(kb, sk, kt.tile(0) * E::BK);
  lv.issue(vb, sv, kt.tile(0) * E::BK);
  RowBits<E::BK> rb(mask, a.N);
  rb.fetch(kt.tile(0) * E::BK);
  if (REL) {
    stage_edges(a.rel, edge);
    __syncthreads();
    build_rel_lut(a, h, edge, lut);
  }

  const int i0 = qt * WIN_RES + wave * 32, t0 = i0 + shift, i = i0 + (lane & 31), t = i + shift;
  const bool row_ok = i < a.M && (!mask || mask[t] != 0.f);
  typename E::Frag qf;
  E::template load_frag<FAST>(
      qf, row_ok ? reinterpret_cast<const T*>(a.q) + b * a.qsb + h * a.qsh + (size_t)i * a.qsn : nullptr, a.d, lane);
  const float sc = a.scale * LOG2E;
  // What the backward takes D = do.o from: the weights of the sums are rounded to bf16, and o once more.  Divided by
  // the sum of the rounded weights, and kept in two parts, o gives a D that is off by the weights' roundings times
  // dp - D alone (the errors of sum p~ dp and D sum p~ cancel), where o's own would be as large as ds in rows that
  // few keys take most of or whose values have much in common.  (Training only: 64 us with it, 58 without, at 16 / 4
  // heads of 4096 tokens, d 128, window 1024.)
  const bool rest = sizeof(T) == 2 && a.o_rest && !win_few_keys(a, (qt + 1) * WIN_RES);
  float m = NEG_BIG, l = 0.f, lr = 0.f;
  f32x16 acc[E::NT] = {};

  constexpr uint64_t KEYS = RowBits<E::BK>::ALL;  // all keys of a tile inside and unmasked
  for (int it = 0; it < kt.total; ++it) {
    const int j0 = kt.tile(it) * E::BK, buf = it & 1;
    T *tk = sk + buf * E::TILE, *tv = sv + buf * E::TILE;
    lds_loads_done();
    __syncthreads();  // this tile is there, and the other buffer's products are done
    const uint64_t now = rb.get();
    if (now != KEYS) {
      clear_rows<T, DP>(tk, now);
      clear_rows<T, DP>(tv, now);
      __syncthreads();
    }
    if (it + 1 < kt.total) {
      const int j1 = kt.tile(it + 1) * E::BK;
      lk.issue(kb, sk + (buf ^ 1) * E::TILE, j1);
      lv.issue(vb, sv + (buf ^ 1) * E::TILE, j1);
      rb.fetch(j1);
    }
    if ((now == 0) | vis.none(t0, j0, E::BK)) continue;
    f32x16 y[E::NSUB];
#pragma unroll
    for (int sub = 0; sub < E::NSUB; ++sub) y[sub] = E::template row_product<true>(tk, 32 * sub, qf, lane);
    // log2 of the weights: ya y + yc.  A tile all of whose pairs are visible and get one table value needs no test a
    // pair; else a table value a pair goes into y itself, and what is not visible becomes -inf.
    float ya[E::NSUB], yc[E::NSUB];
    const int far = REL ? rel_far(a.rel, t0, j0, E::BK) : 0;
#pragma unroll
    for (int sub = 0; sub < E::NSUB; ++sub) ya[sub] = sc, yc[sub] = REL && far >= 0 ? lut[far] : 0.f;
    if ((now != KEYS) | !vis.all_near(t0, j0, E::BK) | (far < 0)) {
#pragma unroll
      for (int sub = 0; sub < E::NSUB; ++sub) {
        const int js = j0 + 32 * sub;
        if (REL && far < 0 && !vis.none(t0, js)) {
          const int one = rel_far(a.rel, t0, js);
          if (one >= 0) {
            yc[sub] = lut[one];
          } else {
            const float* p = lut + rel_lut_base(a.rel) + t - js - 4 * h32;
#pragma unroll
            for (int r = 0; r < 16; ++r) y[sub][r] = __builtin_fmaf(y[sub][r], sc, p[-acc_row(r, 0)]);
            ya[sub] = 1.f;
          }
        }
        const unsigned keys = (unsigned)(now >> (32 * sub));
        if (keys != 0xffffffffu || !vis.all_near(t0, js)) {
          const unsigned mine = keys >> (4 * h32);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int j = js + acc_row(r, h32);
            y[sub][r] = (((mine >> acc_row(r, 0)) & 1u) != 0u) & vis.sees(t, j) ? y[sub][r] : -INFINITY;
          }
        }
      }
    }
    float mx = NEG_BIG;
#pragma unroll
    for (int sub = 0; sub < E::NSUB; ++sub) {
      float top = y[sub][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = fmaxf(top, y[sub][r]);
      mx = fmaxf(mx, __builtin_fmaf(top, ya[sub], yc[sub]));
    }
    mx = xor32_pair(mx, true);
    if (__any(mx > m + WIN_SLACK)) {
      const float to = fmaxf(mx, m), al = fast_exp2(m - to);
      m = to;
      l *= al;
      lr *= al;
#pragma unroll
      for (int n = 0; n < E::NT; ++n) acc[n] *= al;
    }
#pragma unroll
    for (int sub = 0; sub < E::NSUB; ++sub) {
      const float c = yc[sub] - m;
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        y[sub][r] = fast_exp2(__builtin_fmaf(y[sub][r], ya[sub], c));
        s += y[sub][r];
      }
      l += s;
      typename E::Prob p;
      E::to_operand(y[sub], p);
      if constexpr (sizeof(T) == 2) {
        if (rest) lr += E::operand_sum(p, 0.f);
      }
      E::template column_product<true>(tv, 32 * sub, p, acc, lane);
    }
  }
  l = xor32_pair(l, false);
  const bool some = row_ok && l > 0.f;
  const float inv = some ? 1.f / l : 0.f;
  lr = xor32_pair(lr, false);
  const float inv_r = some ? 1.f / lr : 0.f;
  if (i < a.M) {
    const size_t row = ((size_t)b * a.H + h) * a.M + i;
    if (a.lse && h32 == 0) a.lse[row] = some ? m + fast_log2(l) : LSE_EMPTY;
    T* o = reinterpret_cast<T*>(a.o) + row * a.d;
#pragma unroll
    for (int n = 0; n < E::NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        f32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = some ? acc[n][r + e] * inv : 0.f;
        store4<T, FAST>(o, 32 * n + acc_row(r, h32), a.d, w);
      }
    if (rest) {
      T* left = reinterpret_cast<T*>(a.o_rest) + row * a.d;
#pragma unroll
      for (int n = 0; n < E::NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          f32x4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = some ? acc[n][r + e] * inv_r - to_f32(from_f32<T>(acc[n][r + e] * inv)) : 0.f;
          store4<T, FAST>(left, 32 * n + acc_row(r, h32), a.d, w);
        }
    }
  }
}

// 16-byte loads: aligned rows of whole chunks.
template <typename T> static bool win_fast(const WinArgs& a, bool bwd) {
  auto al = [](const void* p) { return ((uintptr_t)p & 15u) == 0; };
  auto st = [](long long s) { return ((s * (long long)sizeof(T)) & 15) == 0; };
  bool ok = (a.d * sizeof(T)) % 16 == 0 && al(a.q) && al(a.k) && al(a.v) && al(a.o) && al(a.o_rest);
  ok = ok && st(a.qsb) && st(a.qsh) && st(a.qsn) && st(a.ksb) && st(a.ksh) && st(a.ksn) && st(a.vsb) && st(a.vsh) &&
       st(a.vsn);
  if (bwd) ok = ok && al(a.go) && al(a.dq) && al(a.dk) && al(a.dv);
  return ok;
}
bool window_fast(const WinArgs& a, bool bf16_in, bool bwd) {
  return bf16_in ? win_fast<bf16>(a, bwd) : win_fast<float>(a, bwd);
}

template <typename T, int DP, bool FAST, bool REL>
static hipError_t fwd_launch(const WinArgs& a, hipStream_t s) {
  using E = WinEng<T, DP>;
  const size_t lds = 4 * E::TILE * sizeof(T) + (REL ? (rel_lut_size(a.rel) + REL_EDGES) * 4 : 0);
  auto kern = window_fwd_kernel<T, DP, FAST, REL>;
  const hipError_t attr = set_lds_limit((const void*)kern, lds);
  if (attr != hipSuccess) return attr;
  const int nqt = (a.M + WIN_RES - 1) / WIN_RES;
  hipLaunchKernelGGL(kern, dim3((unsigned)(nqt * a.B * a.H)), dim3(WIN_NT), lds, s, a);
  return hipGetLastError();
}
template <typename T, int DP> static hipError_t fwd_pick(const WinArgs& a, hipStream_t s) {
  const bool fast = win_fast<T>(a, false);
  if (a.table) return fast ? fwd_launch<T, DP, true, true>(a, s) : fwd_launch<T, DP, false, true>(a, s);
  return fast ? fwd_launch<T, DP, true, false>(a, s) : fwd_launch<T, DP, false, false>(a, s);
}
hipError_t launch_window_fwd(const WinArgs& a, bool bf16_in, int DP, hipStream_t s) {
  if (bf16_in)
    return DP == 32 ? fwd_pick<bf16, 32>(a, s) : DP == 64 ? fwd_pick<bf16, 64>(a, s) : fwd_pick<bf16, 128>(a, s);
  return DP == 32 ? fwd_pick<float, 32>(a, s) : DP == 64 ? fwd_pick<float, 64>(a, s) : fwd_pick<float, 128>(a, s);
}

}  // namespace dfl
