// Attention over a sliding window and a few first tokens, backward (notation of window_attn.hip):
//   p_ij = exp2(y_ij - lse_i), dp_ij = do_i.v_j, D_i = sum_j p_ij dp_ij = do_i.o_i,
//   ds_ij = p_ij (dp_ij - D_i),
//   dq_i = scale sum_j ds_ij k_j, dk_j = scale sum_i ds_ij q_i, dv_j = sum_i p_ij do_i,
//   dtable[h, b] = sum of ds_ij over the pairs of bucket b.
// A query-resident pass gives D, dq and the table's gradient, a key-resident pass dk and dv (summed over the
// query heads of a key head in its registers), so no result passes through an atomic and every sum has one order.
// The first tokens' keys, which all queries see, would make their key tile as long as the sequence: what they get
// from outside the band is summed per query chunk in workgroups of its own and joined by the finalize kernel.
#include "window_engine.h"
#include "window_stage.h"

#include <algorithm>

namespace dfl {

// D_i.  Tiles of queries that see at most WIN_EXACT_KEYS keys each take it as the sum of p dp in a pass of its own over
// them (two products more), so that it holds no rounding of the stored o: where a row has few keys, o's rounding would
// be as large in ds as ds itself.  With more keys fp32 takes do.o and bf16 do.(o + o_rest), see the forward: 74 us
// against 115 with the pass at 16 / 4 heads of 4096 tokens, d 128, window 1024.  Without o_rest bf16 has the pass.
template <typename T, int DP>
__device__ __forceinline__ float frag_dot(const typename WinEng<T, DP>::Frag& x,
                                          const typename WinEng<T, DP>::Frag& y) {
  using E = WinEng<T, DP>;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < E::STEPS; ++i) {
    T a[E::VEC], b[E::VEC];
    __builtin_memcpy(a, &x.v[i], 16);
    __builtin_memcpy(b, &y.v[i], 16);
#pragma unroll
    for (int e = 0; e < E::VEC; ++e) s = __builtin_fmaf(to_f32(a[e]), to_f32(b[e]), s);
  }
  return xor32_pair(s, false);
}

template <typename T, int DP, bool FAST, bool REL>
__global__ void __launch_bounds__(WIN_NT, sizeof(T) == 4 && DP == 128 ? 1 : 2)
    window_bwd_q_kernel(WinArgs a, int n_buf) {
  using E = WinEng<T, DP>;
  extern __shared__ __align__(16) unsigned char smem[];
  T* sk = reinterpret_cast<T*>(smem);  // [n_buf] key tiles, [n_buf] value tiles
  T* sv = sk + n_buf * E::TILE;
  float* lut = reinterpret_cast<float*>(sv + n_buf * E::TILE);
  int* edge = reinterpret_cast<int*>(lut + (REL ? rel_lut_size(a.rel) : 0));
  // The table's gradient: sums of ds by distance, one row of them a wave (every address has one writer), and where a
  // wave turns the diagonals of its pairs into columns.
  const bool tab = REL && a.dtable;
  const int lutn = REL ? rel_lut_size(a.rel) : 0;
  float* hist = reinterpret_cast<float*>(edge + (REL ? REL_EDGES : 0));  // [4][lutn]
  float* skew = hist + (tab ? 4 * lutn : 0);                              // [4][16][64]
  float* far_sums = skew + (tab ? 4 * 16 * 64 : 0);                       // [4][2]
  const int lane = threadIdx.x & 63, h32 = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // uniform: tile tests are scalar

  const int G = a.H / a.Hk, nqt = (a.M + WIN_RES - 1) / WIN_RES;
  int x = xcd_order(blockIdx.x, gridDim.x);
  const int g = x % G;
  x /= G;
  const int qt = x % nqt, bhk = x / nqt, b = bhk / a.Hk, hk = bhk % a.Hk, h = hk * G + g;
  const int shift = a.N - a.M;
  const T* kb = reinterpret_cast<const T*>(a.k) + b * a.ksb + hk * a.ksh;
  const T* vb = reinterpret_cast<const T*>(a.v) + b * a.vsb + hk * a.vsh;
  const float* mask = a.mask ? a.mask + (size_t)b * a.N : nullptr;
  const WinVis vis(a);
  const KeyTiles kt(a, qt * WIN_RES + shift, min(a.M, (qt + 1) * WIN_RES) - 1 + shift, E::BK);
  const RowLoader<T, DP, FAST> lk(a.ksn, a.N, a.d), lv(a.vsn, a.N, a.d);
  RowBits<E::BK> rb(mask, a.N);
  constexpr uint64_t KEYS = RowBits<E::BK>::ALL;
  // Two buffers, the next tile on its way during this one's products; one where a long table's sums take their room.
  auto issue = [&](int it, int buf) {
    const int j0 = kt.tile(it) * E::BK;
    lk.issue(kb, sk + buf * E::TILE, j0);
    lv.issue(vb, sv + buf * E::TILE, j0);
    rb.fetch(j0);
  };
  if (n_buf > 1) issue(0, 0);
  if (REL) {
    stage_edges(a.rel, edge);
    __syncthreads();
    build_rel_lut(a, h, edge, lut);
  }
  if (tab)
    for (int n = threadIdx.x; n < 4 * lutn + 4 * 16 * 64; n += WIN_NT) hist[n] = 0.f;  // (skew behind it)

  const int i0 = qt * WIN_RES + wave * 32, t0 = i0 + shift, i = i0 + (lane & 31), t = i + shift;
  const bool row_ok = i < a.M && (!mask || mask[t] != 0.f);
  const size_t row = ((size_t)b * a.H + h) * a.M + i;
  typename E::Frag qf, gf;
  E::template load_frag<FAST>(
      qf, row_ok ? reinterpret_cast<const T*>(a.q) + b * a.qsb + h * a.qsh + (size_t)i * a.qsn : nullptr, a.d, lane);
  E::template load_frag<FAST>(gf, row_ok ? reinterpret_cast<const T*>(a.go) + row * a.d : nullptr, a.d, lane);
  const float sc = a.scale * LOG2E;
  const float lse = row_ok ? a.lse[row] : LSE_EMPTY;
  const bool exact = win_few_keys(a, (qt + 1) * WIN_RES) || (sizeof(T) == 2 && !a.o_rest);
  float D = 0.f, f = 1.f;
  if (!exact) {
    typename E::Frag of;
    E::template load_frag<FAST>(of, row_ok ? reinterpret_cast<const T*>(a.o) + row * a.d : nullptr, a.d, lane);
    D = frag_dot<T, DP>(of, gf);
    if constexpr (sizeof(T) == 2) {
      E::template load_frag<FAST>(of, row_ok ? reinterpret_cast<const T*>(a.o_rest) + row * a.d : nullptr, a.d, lane);
      D += frag_dot<T, DP>(of, gf);
    }
  }

  // body(p, dp, js) for every 32 x 32 pair that the wave sees something of; `buf`: where the first tile is or goes
  auto sweep = [&](auto body, int& buf, bool again) {
    for (int it = 0; it < kt.total; ++it, buf ^= n_buf - 1) {
      const int j0 = kt.tile(it) * E::BK;
      T *tk = sk + buf * E::TILE, *tv = sv + buf * E::TILE;
      if (n_buf == 1) {
        __syncthreads();
        issue(it, 0);
      }
      lds_loads_done();
      __syncthreads();  // this tile is there, and the other buffer's products are done
      const uint64_t now = rb.get();
      if (now != KEYS) {
        clear_rows<T, DP>(tk, now);
        clear_rows<T, DP>(tv, now);
        __syncthreads();
      }
      if (n_buf > 1 && (it + 1 < kt.total || again)) issue(it + 1 < kt.total ? it + 1 : 0, buf ^ 1);
      if (now == 0) continue;
#pragma unroll
      for (int sub = 0; sub < E::NSUB; ++sub) {
        const int js = j0 + 32 * sub;
        if (vis.none(t0, js)) continue;
        f32x16 y = E::row_product(tk, 32 * sub, qf, lane);
        f32x16 dp = E::row_product(tv, 32 * sub, gf, lane);
        const int far = REL ? rel_far(a.rel, t0, js) : 0;
        if (REL && far < 0) {
          const float* p = lut + rel_lut_base(a.rel) + t - js - 4 * h32;
#pragma unroll
          for (int r = 0; r < 16; ++r) y[r] = __builtin_fmaf(y[r], sc, p[-acc_row(r, 0)]) - lse;
        } else {
          const float c = REL ? lut[far] - lse : -lse;
#pragma unroll
          for (int r = 0; r < 16; ++r) y[r] = __builtin_fmaf(y[r], sc, c);
        }
        const unsigned keys = (unsigned)(now >> (32 * sub));
        if (keys != 0xffffffffu || !vis.all_near(t0, js)) {
          const unsigned mine = keys >> (4 * h32);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int j = js + acc_row(r, h32);
            y[r] = (((mine >> acc_row(r, 0)) & 1u) != 0u) & vis.sees(t, j) ? y[r] : -INFINITY;
          }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) y[r] = fast_exp2(y[r]);
        body(y, dp, js, far, tk, sub);
      }
    }
  };

  int buf = 0;
  if (exact) {
    float sum = 0.f, sdp = 0.f, top = 0.f, next = 0.f;  // next: the second largest weight
    sweep(
        [&](const f32x16& p, const f32x16& dp, int, int, T*, int) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            sum += p[r];
            sdp = __builtin_fmaf(p[r], dp[r], sdp);
            next = __builtin_amdgcn_fmed3f(p[r], top, next);
            top = fmaxf(top, p[r]);
          }
        },
        buf, true);
    sum = xor32_pair(sum, false);
    sdp = xor32_pair(sdp, false);
    next = fmaxf(xor32_pair(next, true), -xor32_pair(-top, true));  // the lane pair's smaller top is a candidate
    // a row with one key has no score gradient; its rounding errors are none either
    f = (sum > 0.f && next == 0.f) ? 0.f : 1.f;
    D = (sum > 0.f && f != 0.f) ? sdp / sum : 0.f;
  }
  if (i < a.M && h32 == 0) {
    a.rowd[2 * row] = D;
    a.rowd[2 * row + 1] = f;
  }

  f32x16 acc[E::NT] = {};
  float far_past = 0.f, far_next = 0.f;
  sweep(
      [&](f32x16& p, const f32x16& dp, int js, int far, T* tk, int sub) {
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] *= __builtin_fmaf(dp[r], f, -D);
        if (tab) {
          if (far >= 0) {
            float s = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) s += p[r];
            if (far > rel_lut_base(a.rel)) far_past += s;
            else far_next += s;
          } else {
            // Key row m and query n lie at distance t0 - js + n - m.  16 rows at a time go to LDS with row m moved by
            // m, so that a column holds one distance: lane x sums column x, distance t0 - js - 16 half - 15 + x.  The
            // entries that no pair belongs to keep the zeros they start with.  (LDS float additions into sums by
            // bucket, 16 a lane and pair, made the pass 61 us instead of 31 at 2 x 16 heads of 1021 tokens.)
            float* sw = skew + wave * 16 * 64;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float* to = sw + (4 * h32) * 64 + (lane & 31) - 4 * h32 + 15;
              wave_lds_fence();  // the last half's columns are read, its sums written
#pragma unroll
              for (int r = 0; r < 8; ++r) to[acc_row(r, 0) * 63] = p[8 * half + r];
              wave_lds_fence();  // a column is other lanes' entries
              float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int m = 0; m < 16; ++m) s[m & 3] += sw[m * 64 + lane];
              float* at = hist + wave * lutn + rel_lut_base(a.rel) + t0 - js - 16 * half - 15 + lane;
              if (lane < 47) *at += (s[0] + s[1]) + (s[2] + s[3]);
            }
          }
        }
        typename E::Prob o;
        E::to_operand(p, o);
        E::column_product(tk, 32 * sub, o, acc, lane);
      },
      buf, false);
  if (i < a.M) {
    T* dq = reinterpret_cast<T*>(a.dq) + row * a.d;
#pragma unroll
    for (int n = 0; n < E::NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        f32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = acc[n][r + e] * a.scale;
        store4<T, FAST>(dq, 32 * n + acc_row(r, h32), a.d, w);
      }
  }
  if (tab) {
    const int nb = a.rel.buckets();
    far_past = wave_sum(far_past);
    far_next = wave_sum(far_next);
    if (lane == 0) far_sums[2 * wave] = far_past, far_sums[2 * wave + 1] = far_next;
    __syncthreads();
    float* part = a.tab_part + (((size_t)b * a.H + h) * nqt + qt) * nb;
    const int base = rel_lut_base(a.rel), ne = a.rel.n;
    for (int n = wave; n < nb; n += WIN_NT / 64) {
      // distances mag of bucket n, [lo, hi), at base + mag (past) or base - mag (future)
      const int k = n <= ne ? n : n - ne - 1, lo = k ? edge[k - 1] : (n <= ne ? 0 : 1);
      const int hi = k < ne ? edge[k] : (n <= ne ? lutn - base : base + 1);
      float s = 0.f;
      for (int mag = lo + lane; mag < hi; mag += 64) {
        const float* at = hist + (n <= ne ? base + mag : base - mag);
        s += (at[0] + at[lutn]) + (at[2 * lutn] + at[3 * lutn]);
      }
      s = wave_sum(s);
      if (k == ne) {
        const float* f4 = far_sums + (n <= ne ? 0 : 1);
        s += (f4[0] + f4[2]) + (f4[4] + f4[6]);
      }
      if (lane == 0) part[n] = s;
    }
  }
}

// Key-resident pass: 64 keys of a (sample, key head) against the queries of their band, 64 staged queries at a time.
// Wave (kg, half) forms p and ds of 32 keys (group kg) and 32 of the staged queries (`half`), and sums one result over
// all of them: half 0 dv, half 1 dk.  So each hands the other half one operand through LDS (p or ds, in bf16 for bf16)
// and keeps one accumulator, not two: 256 registers a lane and two workgroups a CU, where both sums in every wave took
// 474 registers and left each matrix instruction's latency uncovered (196 us against 171 at 16 / 4 heads of 4096 tokens,
// d 128, window 1024, one workgroup a key tile; 146 with two, kv_split).  What bounds it now is the mix of a step: 32
// matrix instructions, 250 others and two barriers a wave, at two waves a SIMD about half of the time in none.
// SINK: 64 of the first tokens' keys against a chunk of the queries outside their band.
constexpr int WIN_KEYS = 64;

template <typename T, int DP, bool FAST, bool REL, bool SINK>
__device__ __forceinline__ void bwd_kv(const WinArgs& a, int x, int n_buf, unsigned char* smem) {
  using E = WinEng<T, DP>;
  constexpr int NB = 64 / E::BK;  // LDS tiles of the engine's size in 64 rows
  constexpr int TILE = 64 * DP;
  T* sq = reinterpret_cast<T*>(smem);  // [n_buf] query tiles, [n_buf] tiles of their output's gradient
  T* sg = sq + n_buf * TILE;
  typename E::Prob* xch = reinterpret_cast<typename E::Prob*>(sg + n_buf * TILE);  // [kg][half][64]: operands
  float* srow = reinterpret_cast<float*>(xch + 4 * 64);                            // [2][3][64]: lse, D, factor
  float* lut = srow + 2 * 3 * 64;
  int* edge = reinterpret_cast<int*>(lut + (REL ? rel_lut_size(a.rel) : 0));
  const int lane = threadIdx.x & 63, h32 = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // uniform: tile tests are scalar
  const int G = a.H / a.Hk, shift = a.N - a.M, kg = wave & 1, half = wave >> 1;
  const WinVis vis(a);

  int bhk, j0, c = 0, sp = 0;
  if (SINK) {
    const int ngrp = (min(a.n_sink, a.N) + WIN_KEYS - 1) / WIN_KEYS;
    c = x % a.n_chunks;
    x /= a.n_chunks;
    j0 = WIN_KEYS * (x % ngrp) + 32 * kg;
    bhk = x / ngrp;
  } else {
    const int nkt = (a.N + WIN_KEYS - 1) / WIN_KEYS;
    sp = x % a.kv_split;
    x /= a.kv_split;
    j0 = (x % nkt) * WIN_KEYS + 32 * kg;
    bhk = x / nkt;
  }
  const int b = bhk / a.Hk, hk = bhk % a.Hk, j = j0 + (lane & 31);
  const float* mask = a.mask ? a.mask + (size_t)b * a.N : nullptr;

  int ilo, ihi;  // queries [ilo, ihi)
  if (SINK) {
    const int first = a.causal ? max(0, min(a.window, a.N) - shift) : 0;
    ilo = first + c * a.chunk;
    ihi = min(a.M, ilo + a.chunk);
  } else {
    const int k0 = j0 - 32 * kg, k1 = min(a.N, k0 + WIN_KEYS) - 1;
    ilo = max(0, k0 - vis.off - shift);
    ihi = min(a.M, k1 - vis.off + (int)vis.range - shift);
  }
  // (head, query tile) pairs, this workgroup's part of them [it0, it1)
  const int nt = ihi > ilo ? (ihi - ilo + 63) / 64 : 0, all = G * nt;
  const int it0 = SINK ? 0 : (int)((long long)all * sp / a.kv_split);
  const int it1 = SINK ? all : (int)((long long)all * (sp + 1) / a.kv_split);
  const RowLoader<T, DP, FAST> lq(a.qsn, a.M, a.d), lg(a.d, a.M, a.d);
  RowBits<64> rb(mask ? mask + shift : nullptr, a.M);
  float r_lse, r_d, r_f;  // of the next tile's row threadIdx.x
  auto issue = [&](int it, int buf) {
    const int h = hk * G + it / nt, i0 = ilo + it % nt * 64;
    const size_t row0 = ((size_t)b * a.H + h) * a.M;
    const T* qb = reinterpret_cast<const T*>(a.q) + b * a.qsb + h * a.qsh;
    const T* gb = reinterpret_cast<const T*>(a.go) + row0 * a.d;
    rb.fetch(i0);
    if (threadIdx.x < 64) {
      const int i = i0 + threadIdx.x;
      const bool ok = i < ihi;
      const size_t at = row0 + min(i, a.M - 1);
      r_lse = ok ? a.lse[at] : LSE_EMPTY;
      r_d = ok ? a.rowd[2 * at] : 0.f;
      r_f = ok ? a.rowd[2 * at + 1] : 0.f;
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      lq.issue(qb, sq + buf * TILE + n * E::TILE, i0 + n * E::BK);
      lg.issue(gb, sg + buf * TILE + n * E::TILE, i0 + n * E::BK);
    }
  };
  auto put_rows = [&](int buf) {
    if (threadIdx.x < 64) {
      float* r = srow + buf * 192 + threadIdx.x;
      r[0] = r_lse;
      r[64] = r_d;
      r[128] = r_f;
    }
  };
  if (REL) stage_edges(a.rel, edge);
  if (n_buf > 1 && it0 < it1) {
    issue(it0, 0);
    put_rows(0);
  }

  const bool key_ok = j < (SINK ? min(a.n_sink, a.N) : a.N) && (!mask || mask[j] != 0.f);
  typename E::Frag kf, vf;
  E::template load_frag<FAST>(
      kf, key_ok ? reinterpret_cast<const T*>(a.k) + b * a.ksb + hk * a.ksh + (size_t)j * a.ksn : nullptr, a.d, lane);
  E::template load_frag<FAST>(
      vf, key_ok ? reinterpret_cast<const T*>(a.v) + b * a.vsb + hk * a.vsh + (size_t)j * a.vsn : nullptr, a.d, lane);
  const float sc = a.scale * LOG2E;
  const int ns = min(a.n_sink, a.N);
  f32x16 acc[E::NT] = {};  // half 0: dv, half 1: dk
  // whether any of the wave's keys and the 32 queries from t0 on meet here
  auto meet = [&](int t0) { return SINK ? (j0 < ns) & vis.some_first(t0, j0) : !vis.none_near(t0, j0); };
  for (int it = it0; it < it1; ++it) {
    const int buf = (it - it0) & (n_buf - 1);
    const bool new_head = REL && (it == it0 || it % nt == 0);
    if (n_buf == 1) {
      __syncthreads();
      issue(it, 0);
      put_rows(0);
    }
    lds_loads_done();
    __syncthreads();  // this tile is there, and the other buffer's products are done
    const uint64_t now = rb.get();
    if (now != ~0ull) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        clear_rows<T, DP>(sq + buf * TILE + n * E::TILE, now >> (n * E::BK & 63));
        clear_rows<T, DP>(sg + buf * TILE + n * E::TILE, now >> (n * E::BK & 63));
      }
      // a masked query's row may have an lse of any value
      if (threadIdx.x < 64 && !((now >> threadIdx.x) & 1u)) srow[buf * 192 + threadIdx.x] = LSE_EMPTY;
    }
    if (new_head) build_rel_lut(a, hk * G + it / nt, edge, lut);
    if (now != ~0ull || new_head) __syncthreads();
    const bool next = n_buf > 1 && it + 1 < it1;
    if (next) issue(it + 1, buf ^ 1);

    const int tile0 = ilo + it % nt * 64 + shift, t0 = tile0 + 32 * half;
    T *tq = sq + buf * TILE, *tg = sg + buf * TILE;
    if (meet(t0)) {
      f32x16 p = E::row_product(tq, 32 * half, kf, lane);
      f32x16 ds = E::row_product(tg, 32 * half, vf, lane);
      const float* sr = srow + buf * 192 + 32 * half + 4 * h32;
      const int far = REL ? rel_far(a.rel, t0, j0) : 0;
      if (REL && far < 0) {
        const float* lp = lut + rel_lut_base(a.rel) + t0 + 4 * h32 - j;
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] = __builtin_fmaf(p[r], sc, lp[acc_row(r, 0)] - sr[acc_row(r, 0)]);
      } else {
        const float cst = REL ? lut[far] : 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] = __builtin_fmaf(p[r], sc, cst - sr[acc_row(r, 0)]);
      }
      if (SINK || !vis.all_near(t0, j0)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int t = t0 + acc_row(r, h32);
          const bool near = vis.near(t, j);
          p[r] = (SINK ? !near & vis.first(t, j) : near) ? p[r] : -INFINITY;
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int at = acc_row(r, 0);
        p[r] = fast_exp2(p[r]);
        ds[r] = p[r] * __builtin_fmaf(ds[r], sr[128 + at], -sr[64 + at]);
      }
      typename E::Prob o, other;
      E::to_operand(half ? ds : p, o);
      E::to_operand(half ? p : ds, other);
      xch[(2 * kg + half) * 64 + lane] = other;
      E::column_product(half ? tq : tg, 32 * half, o, acc, lane);
    }
    lds_barrier();
    if (meet(tile0 + 32 * (half ^ 1))) {
      const typename E::Prob o = xch[(2 * kg + (half ^ 1)) * 64 + lane];
      E::column_product(half ? tq : tg, 32 * (half ^ 1), o, acc, lane);
    }
    if (next) put_rows(buf ^ 1);
  }
  if (j >= (SINK ? ns : a.N)) return;
  const int which = half ? 0 : 1;  // dk before dv in a partial row
  float* part = nullptr;           // joined by the finalize kernel: parts of the queries, the first tokens' rows
  if (!SINK && a.kv_split > 1)
    part = a.kv_part + (((size_t)sp * a.B * a.Hk + bhk) * a.N + j) * 2 * DP + which * DP;
  else if (a.n_chunks > 0 && j < ns)
    part = a.sink_part + (((size_t)bhk * (a.n_chunks + 1) + (SINK ? c : a.n_chunks)) * ns + j) * 2 * DP + which * DP;
  T* out = reinterpret_cast<T*>(half ? a.dk : a.dv) + ((size_t)bhk * a.N + j) * a.d;
  const float f = key_ok ? (half ? a.scale : 1.f) : 0.f;
#pragma unroll
  for (int n = 0; n < E::NT; ++n)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int col = 32 * n + acc_row(r, h32);
      f32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = part ? acc[n][r + e] : key_ok ? acc[n][r + e] * f : 0.f;
      if (part) *reinterpret_cast<f32x4*>(part + col) = w;
      else store4<T, FAST>(out, col, a.d, w);
    }
}

template <typename T, int DP, bool FAST, bool REL>
__global__ void __launch_bounds__(WIN_NT, sizeof(T) == 4 && DP == 128 ? 1 : 2)
    window_bwd_kv_kernel(WinArgs a, int n_sink_blocks, int n_buf) {
  extern __shared__ __align__(16) unsigned char smem[];
  if ((int)blockIdx.x < n_sink_blocks)
    bwd_kv<T, DP, FAST, REL, true>(a, blockIdx.x, n_buf, smem);
  else
    bwd_kv<T, DP, FAST, REL, false>(a, xcd_order(blockIdx.x - n_sink_blocks, gridDim.x - n_sink_blocks), n_buf,
                                       smem);
}

// Rows of dk and dv from their partial sums (parts of the band's queries in order, then the first tokens' chunks),
// and the table's gradient from the query tiles'; a wave for 64 entries of a row or for one table entry, each sum in
// a fixed order.
template <typename T, int DP>
__global__ void __launch_bounds__(WIN_NT) window_finalize_kernel(WinArgs a, int n_row_waves, int n_tab_waves) {
  const int lane = threadIdx.x & 63;
  int w = blockIdx.x * (WIN_NT / 64) + (threadIdx.x >> 6);
  const int ns = min(a.n_sink, a.N), rows = a.kv_split > 1 ? a.N : ns;
  if (w < n_row_waves) {
    const int per = 2 * DP / 64, part = w % per;
    w /= per;
    const int j = w % rows, bhk = w / rows, e = part * 64 + lane, col = e % DP;
    float s = 0.f;
    if (a.kv_split > 1)
      s = ordered_sum(a.kv_part + ((size_t)bhk * a.N + j) * 2 * DP + e, (size_t)a.B * a.Hk * a.N * 2 * DP,
                      a.kv_split, 0.f);
    if (a.n_chunks > 0 && j < ns)  // (without a split the last chunk is the band's)
      s = ordered_sum(a.sink_part + ((size_t)bhk * (a.n_chunks + 1) * ns + j) * 2 * DP + e, (size_t)ns * 2 * DP,
                      a.n_chunks + (a.kv_split == 1), s);
    const bool ok = !a.mask || a.mask[(size_t)(bhk / a.Hk) * a.N + j] != 0.f;
    T* out = reinterpret_cast<T*>(e < DP ? a.dk : a.dv) + ((size_t)bhk * a.N + j) * a.d;
    if (col < a.d) out[col] = from_f32<T>(ok ? (e < DP ? s * a.scale : s) : 0.f);
    return;
  }
  w -= n_row_waves;
  if (w >= n_tab_waves) return;
  const int nb = a.rel.buckets(), h = w / nb, n = w % nb, nqt = (a.M + WIN_RES - 1) / WIN_RES;
  float s = 0.f;
  for (int e = lane; e < a.B * nqt; e += 64) s += a.tab_part[(((size_t)(e / nqt) * a.H + h) * nqt + e % nqt) * nb + n];
  s = wave_sum(s);
  if (lane == 0) a.dtable[w] = s;
}

bool window_fast(const WinArgs& a, bool bf16_in, bool bwd);

template <typename T, int DP, bool FAST, bool REL>
static hipError_t bwd_launch(const WinArgs& a, hipStream_t s) {
  using E = WinEng<T, DP>;
  const size_t lutn = REL ? rel_lut_size(a.rel) : 0, rel = REL ? (lutn + REL_EDGES) * 4 : 0;
  const bool tab = REL && a.dtable;
  const size_t lq1 = rel + (tab ? (4 * lutn + 4 * 16 * 64 + 8) * 4 : 0), buf = 2 * E::TILE * sizeof(T);
  const int n_buf = lq1 + 2 * buf <= 160 * 1024 ? 2 : 1;
  const size_t lq = lq1 + n_buf * buf;
  const size_t lkv1 = 4 * 64 * sizeof(typename E::Prob) + 2 * 3 * 64 * 4 + rel, kbuf = 2 * 64 * DP * sizeof(T);
  const int n_kbuf = lkv1 + 2 * kbuf <= 160 * 1024 ? 2 : 1;
  const size_t lkv = lkv1 + n_kbuf * kbuf;
  auto kq = window_bwd_q_kernel<T, DP, FAST, REL>;
  auto kkv = window_bwd_kv_kernel<T, DP, FAST, REL>;
  hipError_t e = set_lds_limit((const void*)kq, lq);
  if (e != hipSuccess) return e;
  if ((e = set_lds_limit((const void*)kkv, lkv)) != hipSuccess) return e;
  const int nqt = (a.M + WIN_RES - 1) / WIN_RES, nkt = (a.N + WIN_KEYS - 1) / WIN_KEYS, ns = std::min(a.n_sink, a.N);
  hipLaunchKernelGGL(kq, dim3((unsigned)(nqt * a.B * a.H)), dim3(WIN_NT), lq, s, a, n_buf);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  const int nsb = a.n_chunks > 0 ? a.B * a.Hk * a.n_chunks * ((ns + WIN_KEYS - 1) / WIN_KEYS) : 0;
  hipLaunchKernelGGL(kkv, dim3((unsigned)(nkt * a.B * a.Hk * a.kv_split + nsb)), dim3(WIN_NT), lkv, s, a, nsb, n_kbuf);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  const int rows = (a.kv_split > 1 ? a.N : a.n_chunks > 0 ? ns : 0) * a.B * a.Hk * (2 * DP / 64);
  const int tabs = tab ? a.H * a.rel.buckets() : 0;
  if (rows + tabs > 0) {
    hipLaunchKernelGGL((window_finalize_kernel<T, DP>), dim3((unsigned)((rows + tabs + 3) / 4)), dim3(WIN_NT), 0, s, a,
                       rows, tabs);
    e = hipGetLastError();
  }
  return e;
}
template <typename T, int DP> static hipError_t bwd_pick(const WinArgs& a, bool fast, hipStream_t s) {
  if (a.table) return fast ? bwd_launch<T, DP, true, true>(a, s) : bwd_launch<T, DP, false, true>(a, s);
  return fast ? bwd_launch<T, DP, true, false>(a, s) : bwd_launch<T, DP, false, false>(a, s);
}
hipError_t launch_window_bwd(const WinArgs& a, bool bf16_in, int DP, hipStream_t s) {
  const bool fast = window_fast(a, bf16_in, true);
  if (bf16_in)
    return DP == 32   ? bwd_pick<bf16, 32>(a, fast, s)
           : DP == 64 ? bwd_pick<bf16, 64>(a, fast, s)
                      : bwd_pick<bf16, 128>(a, fast, s);
  return DP == 32   ? bwd_pick<float, 32>(a, fast, s)
         : DP == 64 ? bwd_pick<float, 64>(a, fast, s)
                    : bwd_pick<float, 128>(a, fast, s);
}

}  // namespace dfl
