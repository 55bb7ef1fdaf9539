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

// Queries a tile of which sees at most this many keys take D_i as the sum of p dp in a pass of its own over them
// (two products more), so that it holds no rounding of the stored o: where a row has few keys, o's rounding would
// be as large in ds as ds itself.  With more keys o is small against v and do.o is as good.
constexpr int WIN_EXACT_KEYS = 256;

template <typename T, int DP>
__device__ __forceinline__ float frag_dot(const typename WinEng<T, DP>::Frag& x, const typename WinEng<T, DP>::Frag& y) {
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
__global__ void __launch_bounds__(WIN_NT) window_bwd_q_kernel(WinArgs a) {
  using E = WinEng<T, DP>;
  extern __shared__ __align__(16) unsigned char smem[];
  T* sk = reinterpret_cast<T*>(smem);
  T* sv = sk + E::TILE;
  float* lut = reinterpret_cast<float*>(sv + E::TILE);
  // sums by bucket, a column for each thread: every address has one writer
  float* hist = lut + (REL ? rel_lut_size(a.rel) : 0);
  const bool tab = REL && a.dtable;
  uint8_t* lutb = reinterpret_cast<uint8_t*>(hist + (tab ? a.rel.buckets() * WIN_NT : 0));
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
  if (REL) build_rel_lut(a, h, lut, tab ? lutb : nullptr);
  if (tab)
    for (int n = 0; n < a.rel.buckets(); ++n) hist[n * WIN_NT + threadIdx.x] = 0.f;

  const int i0 = qt * WIN_RES + wave * 32, t0 = i0 + shift, i = i0 + (lane & 31), t = i + shift;
  const bool row_ok = i < a.M && (!mask || mask[t] != 0.f);
  const size_t row = ((size_t)b * a.H + h) * a.M + i;
  typename E::Frag qf, gf;
  E::template load_frag<FAST>(
      qf, row_ok ? reinterpret_cast<const T*>(a.q) + b * a.qsb + h * a.qsh + (size_t)i * a.qsn : nullptr, a.d, lane);
  E::template load_frag<FAST>(gf, row_ok ? reinterpret_cast<const T*>(a.go) + row * a.d : nullptr, a.d, lane);
  const float sc = a.scale * LOG2E;
  const float lse = row_ok ? a.lse[row] : LSE_EMPTY;

  const KeyTiles kt(a, qt * WIN_RES + shift, min(a.M, (qt + 1) * WIN_RES) - 1 + shift, E::BK);
  float D = 0.f, f = 1.f;
  const RowLoader<T, DP, FAST> lk(kb, a.ksn, a.N, a.d), lv(vb, a.vsn, a.N, a.d);

  uint64_t bits = 0;
  auto stage = [&](int j0) {
    __syncthreads();
    lk.issue(sk, j0);
    lv.issue(sv, j0);
    RowBits<E::BK> rb(mask, a.N);
    rb.fetch(j0);
    lds_loads_done();
    __syncthreads();
    bits = rb.get();
    if (bits != RowBits<E::BK>::ALL) {
      clear_rows<T, DP>(sk, bits);
      clear_rows<T, DP>(sv, bits);
      __syncthreads();
    }
  };
  // p and dp of one 32 x 32 pair of the staged tile; false where the wave sees nothing of it
  auto pair = [&](int sub, int j0, f32x16& y, f32x16& dp) -> bool {
    const int js = j0 + 32 * sub;
    const bool sinks = js < vis.n_sink && (!vis.causal || js <= t0 + 31);
    if (vis.none_near(t0, js) && !sinks) return false;
    y = E::row_product(sk, 32 * sub, qf, lane);
    dp = E::row_product(sv, 32 * sub, gf, lane);
    if (REL) {
      const int far = rel_far(a.rel, t0, js);
      if (far >= 0) {
        const float c = lut[far] - lse;
#pragma unroll
        for (int r = 0; r < 16; ++r) y[r] = __builtin_fmaf(y[r], sc, c);
      } else {
        const float* p = lut + rel_lut_base(a.rel) + t - js - 4 * h32;
#pragma unroll
        for (int r = 0; r < 16; ++r) y[r] = __builtin_fmaf(y[r], sc, p[-acc_row(r, 0)]) - lse;
      }
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) y[r] = __builtin_fmaf(y[r], sc, -lse);
    }
    const unsigned keys = (unsigned)(bits >> (32 * sub));
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
    return true;
  };

  if (kt.total * E::BK <= WIN_EXACT_KEYS) {
    float sum = 0.f, sdp = 0.f, top = 0.f;
    for (int it = 0; it < kt.total; ++it) {
      const int j0 = kt.tile(it) * E::BK;
      stage(j0);
#pragma unroll
      for (int sub = 0; sub < E::NSUB; ++sub) {
        f32x16 p, dp;
        if (!pair(sub, j0, p, dp)) continue;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          sum += p[r];
          sdp = __builtin_fmaf(p[r], dp[r], sdp);
          top = fmaxf(top, p[r]);
        }
      }
    }
    sum = xor32_pair(sum, false);
    sdp = xor32_pair(sdp, false);
    top = xor32_pair(top, true);
    // a row that one key takes whole has no score gradient; its rounding errors are none either
    f = (sum > 0.f && top == sum) ? 0.f : 1.f;
    D = (sum > 0.f && f != 0.f) ? sdp / sum : 0.f;
  } else {
    typename E::Frag of;
    E::template load_frag<FAST>(of, row_ok ? reinterpret_cast<const T*>(a.o) + row * a.d : nullptr, a.d, lane);
    D = frag_dot<T, DP>(of, gf);
  }
  if (i < a.M && h32 == 0) {
    a.rowd[2 * row] = D;
    a.rowd[2 * row + 1] = f;
  }

  f32x16 acc[E::NT] = {};
  float far_past = 0.f, far_next = 0.f;
  for (int it = 0; it < kt.total; ++it) {
    const int j0 = kt.tile(it) * E::BK;
    stage(j0);
#pragma unroll
    for (int sub = 0; sub < E::NSUB; ++sub) {
      f32x16 p, dp;
      if (!pair(sub, j0, p, dp)) continue;
#pragma unroll
      for (int r = 0; r < 16; ++r) p[r] *= __builtin_fmaf(dp[r], f, -D);
      if (tab) {
        const int js = j0 + 32 * sub, far = rel_far(a.rel, t0, js);
        if (far >= 0) {
          float s = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) s += p[r];
          if (far > rel_lut_base(a.rel)) far_past += s;
          else far_next += s;
        } else {
          const uint8_t* lb = lutb + rel_lut_base(a.rel) + t - js - 4 * h32;
#pragma unroll
          for (int r = 0; r < 16; ++r)
            __hip_atomic_fetch_add(hist + lb[-acc_row(r, 0)] * WIN_NT + threadIdx.x, p[r], __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_WORKGROUP);
        }
      }
      typename E::Prob o;
      E::to_operand(p, o);
      E::column_product(sk, 32 * sub, o, acc, lane);
    }
  }
  if (i < a.M) {
    T* dq = reinterpret_cast<T*>(a.dq) + row * a.d;
#pragma unroll
    for (int n = 0; n < E::NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int c = 32 * n + acc_row(r, h32);
        if (c < a.d) dq[c] = from_f32<T>(acc[n][r] * a.scale);
      }
  }
  if (tab) {
    const int nb = a.rel.buckets();
    hist[a.rel.n * WIN_NT + threadIdx.x] += far_past;  // the last bucket of the queries' past ..
    if (a.rel.both) hist[(nb - 1) * WIN_NT + threadIdx.x] += far_next;  // .. and of their future
    __syncthreads();
    float* part = a.tab_part + (((size_t)b * a.H + h) * nqt + qt) * nb;
    for (int n = wave; n < nb; n += WIN_NT / 64) {
      const f32x4 s = *reinterpret_cast<const f32x4*>(hist + n * WIN_NT + 4 * lane);
      const float tot = wave_sum((s[0] + s[1]) + (s[2] + s[3]));
      if (lane == 0) part[n] = tot;
    }
  }
}

// Key-resident pass.  SINK: 32 of the first tokens' keys against a chunk of the queries outside their band, a
// wave 32 of the staged queries at a time; else 128 keys against the queries of their band, a wave 32 of the keys.
template <typename T, int DP, bool FAST, bool REL, bool SINK>
__device__ __forceinline__ void bwd_kv(const WinArgs& a, int x, unsigned char* smem) {
  using E = WinEng<T, DP>;
  T* sq = reinterpret_cast<T*>(smem);
  T* sg = sq + E::TILE;
  float* srow = reinterpret_cast<float*>(sg + E::TILE);  // [3][BK]: lse, D, factor
  float* lut = srow + 3 * E::BK;
  const int lane = threadIdx.x & 63, h32 = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // uniform: tile tests are scalar
  const int G = a.H / a.Hk, shift = a.N - a.M;
  const WinVis vis(a);

  int bhk, j0, c = 0;
  if (SINK) {
    const int ngrp = (min(a.n_sink, a.N) + 31) / 32;
    c = x % a.n_chunks;
    x /= a.n_chunks;
    j0 = 32 * (x % ngrp);
    bhk = x / ngrp;
  } else {
    const int nkt = (a.N + WIN_RES - 1) / WIN_RES;
    j0 = (x % nkt) * WIN_RES + wave * 32;
    bhk = x / nkt;
  }
  const int b = bhk / a.Hk, hk = bhk % a.Hk, j = j0 + (lane & 31);
  const float* mask = a.mask ? a.mask + (size_t)b * a.N : nullptr;
  const bool key_ok = j < (SINK ? min(a.n_sink, a.N) : a.N) && (!mask || mask[j] != 0.f);
  typename E::Frag kf, vf;
  E::template load_frag<FAST>(
      kf, key_ok ? reinterpret_cast<const T*>(a.k) + b * a.ksb + hk * a.ksh + (size_t)j * a.ksn : nullptr, a.d, lane);
  E::template load_frag<FAST>(
      vf, key_ok ? reinterpret_cast<const T*>(a.v) + b * a.vsb + hk * a.vsh + (size_t)j * a.vsn : nullptr, a.d, lane);
  const float sc = a.scale * LOG2E;

  int ilo, ihi;  // queries [ilo, ihi)
  if (SINK) {
    const int first = a.causal ? max(0, min(a.window, a.N) - shift) : 0;
    ilo = first + c * a.chunk;
    ihi = min(a.M, ilo + a.chunk);
  } else {
    const int k0 = j0 - wave * 32, k1 = min(a.N, k0 + WIN_RES) - 1;
    ilo = max(0, k0 - vis.off - shift);
    ihi = min(a.M, k1 - vis.off + (int)vis.range - shift);
  }
  f32x16 dk[E::NT] = {}, dv[E::NT] = {};
  for (int g = 0; g < G; ++g) {
    const int h = hk * G + g;
    if (REL) {
      __syncthreads();
      build_rel_lut(a, h, lut, nullptr);
    }
    const T* qb = reinterpret_cast<const T*>(a.q) + b * a.qsb + h * a.qsh;
    const size_t row0 = ((size_t)b * a.H + h) * a.M;
    const T* gb = reinterpret_cast<const T*>(a.go) + row0 * a.d;
    const RowLoader<T, DP, FAST> lq(qb, a.qsn, a.M, a.d), lg(gb, a.d, a.M, a.d);
    for (int i0 = ilo; i0 < ihi; i0 += E::BK) {
      __syncthreads();
      lq.issue(sq, i0);
      lg.issue(sg, i0);
      RowBits<E::BK> rb(mask ? mask + shift : nullptr, a.M);
      rb.fetch(i0);
      if ((int)threadIdx.x < E::BK) {
        const int i = i0 + threadIdx.x;
        const bool ok = i < ihi && (!mask || mask[shift + i] != 0.f);
        srow[threadIdx.x] = ok ? a.lse[row0 + i] : LSE_EMPTY;
        srow[E::BK + threadIdx.x] = ok ? a.rowd[2 * (row0 + i)] : 0.f;
        srow[2 * E::BK + threadIdx.x] = ok ? a.rowd[2 * (row0 + i) + 1] : 0.f;
      }
      lds_loads_done();
      __syncthreads();
      const uint64_t bits = rb.get();
      if (bits != RowBits<E::BK>::ALL) {
        clear_rows<T, DP>(sq, bits);
        clear_rows<T, DP>(sg, bits);
        __syncthreads();
      }
#pragma unroll
      for (int sub = 0; sub < E::NSUB; ++sub) {
        const int t0 = i0 + 32 * sub + shift;
        if (SINK ? (sub != wave || vis.all_near(t0, j0)) : vis.none_near(t0, j0)) continue;
        f32x16 p = E::row_product(sq, 32 * sub, kf, lane);
        f32x16 ds = E::row_product(sg, 32 * sub, vf, lane);
        if (REL) {
          const int far = rel_far(a.rel, t0, j0);
          if (far >= 0) {
            const float cst = lut[far];
#pragma unroll
            for (int r = 0; r < 16; ++r) p[r] = __builtin_fmaf(p[r], sc, cst);
          } else {
            const float* lp = lut + rel_lut_base(a.rel) + t0 + 4 * h32 - j;
#pragma unroll
            for (int r = 0; r < 16; ++r) p[r] = __builtin_fmaf(p[r], sc, lp[acc_row(r, 0)]);
          }
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) p[r] *= sc;
        }
        if (SINK || !vis.all_near(t0, j0)) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int t = t0 + acc_row(r, h32);
            const bool near = vis.near(t, j);
            p[r] = (SINK ? !near & vis.first(t, j) : near) ? p[r] : -INFINITY;
          }
        }
        const float* sr = srow + 32 * sub + 4 * h32;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int at = acc_row(r, 0);
          p[r] = fast_exp2(p[r] - sr[at]);
          ds[r] = p[r] * __builtin_fmaf(ds[r], sr[2 * E::BK + at], -sr[E::BK + at]);
        }
        typename E::Prob o;
        E::to_operand(p, o);
        E::column_product(sg, 32 * sub, o, dv, lane);
        E::to_operand(ds, o);
        E::column_product(sq, 32 * sub, o, dk, lane);
      }
    }
  }
  const int ns = min(a.n_sink, a.N);
  if (SINK) {
    // the waves' sums meet in LDS, added in wave order
    float* red = reinterpret_cast<float*>(smem);  // [32][2][DP] over the staged tiles
    for (int w = 0; w < E::NSUB; ++w) {
      __syncthreads();
      if (wave != w) continue;
#pragma unroll
      for (int n = 0; n < E::NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float* at = red + (lane & 31) * 2 * DP + 32 * n + acc_row(r, h32);
          at[0] = w ? at[0] + dk[n][r] : dk[n][r];
          at[DP] = w ? at[DP] + dv[n][r] : dv[n][r];
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 32 * 2 * DP; e += WIN_NT) {
      const int r = e / (2 * DP);
      if (j0 + r < ns)
        a.sink_part[(((size_t)bhk * (a.n_chunks + 1) + c) * ns + j0 + r) * 2 * DP + e % (2 * DP)] = red[e];
    }
    return;
  }
  if (j >= a.N) return;
  if (a.n_chunks > 0 && j < ns) {  // joined with the chunks' sums by the finalize kernel
    float* at = a.sink_part + (((size_t)bhk * (a.n_chunks + 1) + a.n_chunks) * ns + j) * 2 * DP;
#pragma unroll
    for (int n = 0; n < E::NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        at[32 * n + acc_row(r, h32)] = dk[n][r];
        at[DP + 32 * n + acc_row(r, h32)] = dv[n][r];
      }
    return;
  }
  const size_t krow = ((size_t)bhk * a.N + j) * a.d;
#pragma unroll
  for (int n = 0; n < E::NT; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int col = 32 * n + acc_row(r, h32);
      if (col < a.d) {
        reinterpret_cast<T*>(a.dk)[krow + col] = from_f32<T>(key_ok ? dk[n][r] * a.scale : 0.f);
        reinterpret_cast<T*>(a.dv)[krow + col] = from_f32<T>(key_ok ? dv[n][r] : 0.f);
      }
    }
}

template <typename T, int DP, bool FAST, bool REL>
__global__ void __launch_bounds__(WIN_NT) window_bwd_kv_kernel(WinArgs a, int n_sink_blocks) {
  extern __shared__ __align__(16) unsigned char smem[];
  if ((int)blockIdx.x < n_sink_blocks)
    bwd_kv<T, DP, FAST, REL, true>(a, blockIdx.x, smem);
  else
    bwd_kv<T, DP, FAST, REL, false>(a, xcd_order(blockIdx.x - n_sink_blocks, gridDim.x - n_sink_blocks), smem);
}

// The first tokens' rows from their partial sums (band last), and the table's gradient from the query tiles'; a wave
// for 64 entries of a row or for one table entry, each sum in a fixed order.
template <typename T, int DP>
__global__ void __launch_bounds__(WIN_NT) window_finalize_kernel(WinArgs a, int n_row_waves, int n_tab_waves) {
  const int lane = threadIdx.x & 63;
  int w = blockIdx.x * (WIN_NT / 64) + (threadIdx.x >> 6);
  const int ns = min(a.n_sink, a.N);
  if (w < n_row_waves) {
    const int per = 2 * DP / 64, part = w % per;
    w /= per;
    const int j = w % ns, bhk = w / ns, e = part * 64 + lane, col = e % DP;
    const float* p = a.sink_part + ((size_t)bhk * (a.n_chunks + 1) * ns + j) * 2 * DP + e;
    const float s = ordered_sum(p, (size_t)ns * 2 * DP, a.n_chunks + 1, 0.f);
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
  const size_t tiles = 2 * E::TILE * sizeof(T), lutn = REL ? rel_lut_size(a.rel) : 0;
  const bool tab = REL && a.dtable;
  const size_t lq = tiles + lutn * 4 + (tab ? a.rel.buckets() * WIN_NT * 4 + lutn : 0);
  // the first tokens' reduction takes 64 DP floats over the tiles
  const size_t lkv = std::max(tiles + 3 * E::BK * 4 + lutn * 4, (size_t)64 * DP * 4);
  auto kq = window_bwd_q_kernel<T, DP, FAST, REL>;
  auto kkv = window_bwd_kv_kernel<T, DP, FAST, REL>;
  hipError_t e = set_lds_limit((const void*)kq, lq);
  if (e != hipSuccess) return e;
  if ((e = set_lds_limit((const void*)kkv, lkv)) != hipSuccess) return e;
  const int nqt = (a.M + WIN_RES - 1) / WIN_RES, nkt = (a.N + WIN_RES - 1) / WIN_RES, ns = std::min(a.n_sink, a.N);
  hipLaunchKernelGGL(kq, dim3((unsigned)(nqt * a.B * a.H)), dim3(WIN_NT), lq, s, a);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  const int nsb = a.n_chunks > 0 ? a.B * a.Hk * a.n_chunks * ((ns + 31) / 32) : 0;
  hipLaunchKernelGGL(kkv, dim3((unsigned)(nkt * a.B * a.Hk + nsb)), dim3(WIN_NT), lkv, s, a, nsb);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  const int rows = a.n_chunks > 0 ? a.B * a.Hk * ns * (2 * DP / 64) : 0, tabs = tab ? a.H * a.rel.buckets() : 0;
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
