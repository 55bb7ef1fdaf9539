// Products of tokens and weights in 8-bit integers: codes and a scale for each token, formed here, codes and a scale for
// each row of the weights, and the exact 32-bit integer sums times both scales.
//
// Bounds: large products the matrix instructions at the clock that they leave (8192 x 4096 x 4096: 130-144 us, 1900-2110 TOP/s,
// where a library's product in 8-bit integers reaches 2150 and the same loop without its loads 2180-2550), the codes memory (19
// us for 100 MB); few tokens the weights' bytes and latency (1 x 4096 x 4096: 5.8-6.2 us, 32: 4.6 + 8.8).
#include "launch_slices.h"
#include "lowbit_args.h"
#include "lowbit_codes.h"

#include <algorithm>
#include <initializer_list>

namespace dfl {

typedef __attribute__((__vector_size__(4 * sizeof(int)))) int i32x4;
typedef __attribute__((__vector_size__(16 * sizeof(int)))) int i32x16;

constexpr float I8_MIN_SCALE = 0x1p-100f;

// The integer nearest to x / s, ties to even: rint(x * (1 / s)) is it or a neighbour, and the remainder x - q s, which
// one fused multiply-add gives exactly, says which (fp32 quotients would round onto a tie now and then).
__device__ __forceinline__ float i8_code(float x, float s, float inv) {
  float q = __builtin_rintf(x * inv);
  const float r = __builtin_fmaf(-q, s, x), half = 0.5f * s;
  const bool odd = ((int)q & 1) != 0;
  if (r > half || (r == half && odd)) q += 1.f;
  if (r < -half || (r == -half && odd)) q -= 1.f;
  return q;
}

// The scale of a row by its largest magnitude's bits: NaN where that is no finite number.
__device__ __forceinline__ float i8_scale(unsigned top) {
  return top < 0x7f800000u ? fmaxf(__uint_as_float(top) / 127.f, I8_MIN_SCALE) : __builtin_nanf("");
}
// 8 codes; zeros where the scale is NaN.
__device__ __forceinline__ void i8_codes(const float (&v)[8], float s, float inv, unsigned (&w)[2]) {
  // 1.5 * 2^23 + x / s, nearly: a code in the low bits, and the right one where the remainder is less than half a step
  unsigned u[8];
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = __builtin_fmaf(v[i], inv, 12582912.f);
    far = fmaxf(far, fabsf(__builtin_fmaf(12582912.f - y, s, v[i])));
    u[i] = __float_as_uint(y);
  }
  w[0] = w[1] = 0u;
  if (s == s) {
    if (far >= 0.5f * s) {
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = (unsigned)(int)i8_code(v[i], s, inv);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) w[h] = low_bytes(u[4 * h], u[4 * h + 1], u[4 * h + 2], u[4 * h + 3]);
  }
}

// A row a workgroup of 64 W threads, its elements in registers where they fit.
constexpr int I8_KEEP = 4;  // 8 elements each
template <typename T, bool FAST, int W> __global__ void __launch_bounds__(64 * W) row_codes_kernel(RowCodesArgs a) {
  __shared__ unsigned s_top[W];
  const size_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.xs;
  int8_t* out = a.codes + row * a.cs;
  float e[I8_KEEP][8];
  unsigned top = 0;
  auto look = [&](const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  };
#pragma unroll
  for (int k = 0; k < I8_KEEP; ++k) {
    load8<T, FAST>(x, threadIdx.x + k * 64 * W, a.K, e[k]);
    look(e[k]);
  }
  for (int c = threadIdx.x + I8_KEEP * 64 * W; c * 8 < a.K; c += 64 * W) {
    float v[8];
    load8<T, FAST>(x, c, a.K, v);
    look(v);
  }
  top = wave_max_u32(top);
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) top = max(top, s_top[w]);
  }
  const float s = i8_scale(top), inv = 1.f / s;
  if (threadIdx.x == 0) a.scale[row] = s;
  auto put = [&](int c, const float (&v)[8]) {
    unsigned w[2];
    i8_codes(v, s, inv, w);
    *reinterpret_cast<uint2*>(out + c * 8) = make_uint2(w[0], w[1]);
  };
#pragma unroll
  for (int k = 0; k < I8_KEEP; ++k) {
    const int c = threadIdx.x + k * 64 * W;
    if ((long long)c * 8 < a.cs) put(c, e[k]);
  }
  for (int c = threadIdx.x + I8_KEEP * 64 * W; (long long)c * 8 < a.cs; c += 64 * W) {
    float v[8];
    load8<T, FAST>(x, c, a.K, v);
    put(c, v);
  }
}

// The sum of a token and a row of weights as a result.
template <typename T> struct I8Out {
  const float* ws;
  const T* bias;
  T* y;
  int N;
  __device__ __forceinline__ explicit I8Out(const Int8LinearArgs& a)
      : ws(a.w_scale), bias(reinterpret_cast<const T*>(a.bias)), y(reinterpret_cast<T*>(a.y)), N(a.N) {}
  __device__ __forceinline__ T value(int sum, float as, float wsn, float bn) const {
    return from_f32<T>(__builtin_fmaf((float)sum * wsn, as, bn));
  }
};

// Few tokens: the weights go by once.  A workgroup has 16 rows of weights and MT tiles of 16 tokens; its waves share K,
// in steps of 128 bytes, straight from memory into the operands: lane l holds row l % 16 and the 32 bytes l / 16 of a step
// (any order of the bytes will do, as long as weights and tokens have the same).
// OWN: each workgroup forms its tokens' codes itself, OWN tokens a wave, while its first weights arrive: one launch, and no
// workspace.  A wave keeps I8_OWN elements: 1 token of 4096, 2 of 2048 or 4 of 1024.
constexpr int I8_OWN = 4096, I8_OWN_N = 12288;
template <typename T, int MT, int OWN, bool FAST> __global__ void __launch_bounds__(512) int8_few_kernel(Int8LinearArgs a) {
  constexpr int WAVES = 8, U = 4;  // steps in flight
  __shared__ int s_sum[WAVES][MT][16][17];
  __shared__ float s_scale[16 * MT];
  extern __shared__ __align__(16) int8_t s_x[];  // OWN: [tokens][steps * 128 + 16] codes
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, h = lane >> 4;
  const int n0 = (a.first + blockIdx.x) * 16, m0 = blockIdx.y * (16 * MT);
  const int8_t* w = a.w + (long long)min(n0 + r, a.N - 1) * a.ws;
  const int steps = (a.K + 127) / 128, tail = ((a.K + 15) & ~15) - 16;  // last 16 bytes of a row of weights
  auto weights = [&](i32x4 (&v)[2], int s) {
    const int k = s * 128 + 32 * h;  // (past the row's end: tokens are zero there)
    v[0] = *reinterpret_cast<const i32x4*>(w + min(k, tail));
    v[1] = *reinterpret_cast<const i32x4*>(w + min(k + 16, tail));
  };
  i32x4 sum[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) sum[i] = i32x4{0, 0, 0, 0};
  if constexpr (OWN) {
    i32x4 wv[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) weights(wv[u], min(wave + u * WAVES, steps - 1));
    // OWN tokens a wave: the largest magnitude, the scale, the codes of each
    constexpr int KEEP = I8_OWN / OWN / (64 * 8);
    const int tokens = min(a.M - m0, 16 * MT), stride = steps * 128 + 16;
    Eight<T> e[OWN][KEEP];
#pragma unroll
    for (int t = 0; t < OWN; ++t) {  // (a wave without a token takes the last one, and stores nothing)
      const T* row = reinterpret_cast<const T*>(a.x) + (m0 + min(wave + t * WAVES, tokens - 1)) * a.xs;
#pragma unroll
      for (int k = 0; k < KEEP; ++k) load8<FAST>(e[t][k], row, lane + 64 * k, a.K);
    }
#pragma unroll
    for (int t = 0; t < OWN; ++t) {
      const int m = wave + t * WAVES;
      if (m >= tokens) continue;
      unsigned top = 0;
#pragma unroll
      for (int k = 0; k < KEEP; ++k) {
        float f[8];
        lb_floats(e[t][k], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
      }
      const float s = i8_scale(wave_max_u32(top)), inv = 1.f / s;
      if (lane == 0) s_scale[m] = s;
#pragma unroll
      for (int k = 0; k < KEEP; ++k) {
        const int c = lane + 64 * k;
        float f[8];
        unsigned q[2];
        lb_floats(e[t][k], f);
        i8_codes(f, s, inv, q);
        if (c < steps * 16) *reinterpret_cast<uint2*>(s_x + m * stride + c * 8) = make_uint2(q[0], q[1]);
      }
    }
    lds_barrier();
    const int8_t* x[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) x[i] = s_x + min(16 * i + r, tokens - 1) * stride + 32 * h;
    for (int s0 = wave; s0 < steps; s0 += WAVES * U) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int s = s0 + u * WAVES;
        if (s < steps) {
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const i32x4* xv = reinterpret_cast<const i32x4*>(x[i] + s * 128);
            sum[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[u][0], xv[0], sum[i], 0, 0, 0);
            sum[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[u][1], xv[1], sum[i], 0, 0, 0);
          }
        }
        if (s + WAVES * U < steps) weights(wv[u], s + WAVES * U);
      }
    }
  } else {
    const int8_t* x[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) x[i] = a.a + (long long)min(m0 + 16 * i + r, a.M - 1) * a.as;
    for (int s0 = wave; s0 < steps; s0 += WAVES * U) {
      i32x4 wv[U][2], xv[U][MT][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int s = min(s0 + u * WAVES, steps - 1);
        weights(wv[u], s);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const i32x4* at = reinterpret_cast<const i32x4*>(x[i] + s * 128 + 32 * h);
          xv[u][i][0] = at[0], xv[u][i][1] = at[1];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s0 + u * WAVES < steps) {
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            sum[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[u][0], xv[u][i][0], sum[i], 0, 0, 0);
            sum[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[u][1], xv[u][i][1], sum[i], 0, 0, 0);
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s_sum[wave][i][r][4 * h + j] = sum[i][j];  // [token][row of weights]
  __syncthreads();
  const I8Out<T> out(a);
  for (int e = threadIdx.x; e < MT * 256; e += 512) {
    const int m = e >> 4, c = e & 15;
    if (m0 + m >= a.M || n0 + c >= a.N) continue;
    int t = 0;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) t += s_sum[v][m >> 4][m & 15][c];
    const float b = out.bias ? to_f32(out.bias[n0 + c]) : 0.f, as = OWN ? s_scale[m] : a.a_scale[m0 + m];
    out.y[(size_t)(m0 + m) * a.N + n0 + c] = out.value(t, as, out.ws[n0 + c], b);
  }
}

// One 16-byte load a lane from `from` to `to` + 16 lane in LDS (`to` uniform, in bytes); waited for by i8_wait.
__device__ __forceinline__ void i8_load_to_lds(const void* from, unsigned to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(to) : "memory", "m0");
}
// All but the latest N of the wave's loads done.
template <int N> __device__ __forceinline__ void i8_wait() {
  static_assert(N < 64, "vmcnt has six bits");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14);
  asm volatile("" ::: "memory");
}

// Tiles of TM tokens and TN rows of weights, WM x WN waves of 32 x 32 blocks.  K goes by in steps of 128 bytes, whole lines
// of memory, through BUF LDS buffers that are loaded without passing through registers; a row's 16-byte chunk c lies
// at position c ^ (row / 2 % 8), so that 16 lanes reading the same chunk of 16 rows meet every bank once.  The weights are
// the instructions' first operand: a lane of the accumulators has one token and runs of four rows of weights, and the results
// leave through LDS in whole lines.
template <typename T, int TM, int TN, int WM, int WN, int BUF>
__global__ void __launch_bounds__(64 * WM * WN) int8_tile_kernel(Int8LinearArgs a) {
  constexpr int NT = 64 * WM * WN, BK = 128, SUB = BK / 32, MI = TM / WM / 32, NI = TN / WN / 32;
  constexpr int CHUNKS = (TM + TN) * 8, PER = CHUNKS / NT, STEP = NT / 8;  // rows between a thread's chunks
  constexpr int TILE = (TM + TN) * BK;
  static_assert(CHUNKS % NT == 0 && STEP % 16 == 0 && TM % STEP == 0, "whole loads of one swizzle");
  extern __shared__ __align__(16) int8_t s_tile[];  // [BUF][TM + TN][128]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // neighbouring tiles on one XCD; within it columns of 8 tiles of tokens, so that few rows of weights are in use at once
  const int mt = (a.M + TM - 1) / TM, nt = (a.N + TN - 1) / TN;
  int at = blockIdx.x;
  {
    const int total = mt * nt, per = total >> 3, rem = total & 7, xcd = at & 7;
    at = xcd * per + min(xcd, rem) + (at >> 3);
  }
  const int band = at / (8 * nt), rows = min(8, mt - band * 8), in = at - band * 8 * nt;
  const int m0 = (band * 8 + in % rows) * TM, n0 = in / rows * TN;

  const int r0 = threadIdx.x >> 3, chunk = (threadIdx.x & 7) ^ ((r0 >> 1) & 7);
  const int8_t* from[PER];
  int last[PER];  // the furthest chunk that a row may be read at
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    const int r = r0 + p * STEP;
    if (p * STEP < TM) {
      from[p] = a.a + (long long)min(m0 + r, a.M - 1) * a.as;
      last[p] = (int)a.as - 16;
    } else {
      from[p] = a.w + (long long)min(n0 + r - TM, a.N - 1) * a.ws;
      last[p] = ((a.K + 15) & ~15) - 16;  // (past the row's end: tokens are zero there)
    }
  }
  const unsigned base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) int8_t*)s_tile;
  const unsigned to = __builtin_amdgcn_readfirstlane(base + (threadIdx.x & ~63u) * 16);
  const int steps = (a.K + BK - 1) / BK;
  auto issue = [&](int step) {
    const int k = min(step, steps - 1) * BK + chunk * 16;
#pragma unroll
    for (int p = 0; p < PER; ++p) i8_load_to_lds(from[p] + min(k, last[p]), to + (step % BUF) * TILE + p * NT * 16);
  };

  i32x16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = i32x16{};
  const int wm = wave / WN, wn = wave % WN, row = lane & 31, hi = lane >> 5;
  const int8_t* xrow = s_tile + (wm * MI * 32 + row) * BK;
  const int8_t* wrow = s_tile + (TM + wn * NI * 32 + row) * BK;
  struct Part {
    i32x4 x[MI], w[NI];
  };
  auto read = [&](Part& f, int step, int kk) {
    const int pos = ((2 * kk + hi) ^ ((row >> 1) & 7)) * 16 + (step % BUF) * TILE;
#pragma unroll
    for (int i = 0; i < MI; ++i) f.x[i] = *reinterpret_cast<const i32x4*>(xrow + i * 32 * BK + pos);
#pragma unroll
    for (int j = 0; j < NI; ++j) f.w[j] = *reinterpret_cast<const i32x4*>(wrow + j * 32 * BK + pos);
  };
  auto multiply = [&](const Part& f) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[j], f.x[i], acc[i][j], 0, 0, 0);
  };
  // A quarter of a step is read while the one before is multiplied; before the last quarter every wave has read all of
  // its tile, the next one is there, and the buffer is filled anew.  (Left to itself the compiler moves the reads to their
  // use, and waits for each.)
#pragma unroll
  for (int s = 0; s < BUF; ++s) issue(s);
  i8_wait<(BUF - 1) * PER>();
  lds_barrier();
  Part f[2];
  read(f[0], 0, 0);
  for (int s = 0; s < steps; ++s) {
#pragma unroll
    for (int kk = 0; kk < SUB; ++kk) {
      if (kk + 1 < SUB) {
        read(f[(kk + 1) & 1], s, kk + 1);
      } else {
        i8_wait<(BUF - 2) * PER>();
        lds_barrier();
        issue(s + BUF);
        read(f[0], s + 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      multiply(f[kk & 1]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  i8_wait<0>();  // no load is left in flight when the buffers go to the results
  lds_barrier();

  // Results: 32 tokens of the wave at a time, rows of NI * 32 in LDS with the 16-byte chunks exchanged as above.
  constexpr int COLS = NI * 32, RC = COLS * (int)sizeof(T) / 16;  // chunks of a row
  auto place = [](int m, int c) { return (c ^ (RC == 16 ? m & 15 : RC == 8 ? (m >> 1) & 7 : (m >> 2) & 3)) * 16; };
  unsigned char* mine = reinterpret_cast<unsigned char*>(s_tile) + wave * (32 * RC * 16);
  const I8Out<T> out(a);
  const int nw = n0 + wn * COLS;
  const bool whole = ((size_t)a.N * sizeof(T)) % 16 == 0 && ((uintptr_t)a.y & 15) == 0;
  f32x4 ws[NI][4], bias[NI][4];
#pragma unroll
  for (int j = 0; j < NI; ++j)
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = min(nw + j * 32 + 8 * g + 4 * hi + e, a.N - 1);
        ws[j][g][e] = out.ws[n];
        bias[j][g][e] = out.bias ? to_f32(out.bias[n]) : 0.f;
      }
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int mw = m0 + (wm * MI + i) * 32;
    const float as = a.a_scale[min(mw + row, a.M - 1)];
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        T v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = out.value(acc[i][j][4 * g + e], as, ws[j][g][e], bias[j][g][e]);
        const int b = (j * 32 + 8 * g + 4 * hi) * (int)sizeof(T);
        __builtin_memcpy(__builtin_assume_aligned(mine + row * (RC * 16) + place(row, b / 16) + b % 16, sizeof(v)), v, sizeof(v));
      }
    wave_lds_fence();
    if (whole) {
#pragma unroll
      for (int x = 0; x < RC / 2; ++x) {
        const int m = (x * 64 + lane) / RC, c = lane % RC, n = nw + c * (16 / (int)sizeof(T));
        if (mw + m < a.M && n < a.N)
          *reinterpret_cast<i32x4*>(out.y + (size_t)(mw + m) * a.N + n) =
              *reinterpret_cast<const i32x4*>(mine + m * (RC * 16) + place(m, c));
      }
    } else {
      for (int x = 0; x < 32 * COLS / 64; ++x) {
        const int m = (x * 64 + lane) / COLS, n = lane % COLS + (COLS > 64 ? x % (COLS / 64) * 64 : 0), b = n * (int)sizeof(T);
        if (mw + m < a.M && nw + n < a.N)
          out.y[(size_t)(mw + m) * a.N + nw + n] = *reinterpret_cast<const T*>(mine + m * (RC * 16) + place(m, b / 16) + b % 16);
      }
    }
    wave_lds_fence();
  }
}

template <typename T> static bool aligned16(const void* p, std::initializer_list<long long> strides) {
  bool ok = ((uintptr_t)p & 15u) == 0;
  for (long long s : strides) ok = ok && ((s * (long long)sizeof(T)) & 15) == 0;
  return ok;
}
template <typename T, int W> static hipError_t codes_w(const RowCodesArgs& a, hipStream_t s) {
  const bool fast = a.K % 8 == 0 && aligned16<T>(a.x, {a.xs});
  return launch_slices(a.M, 64 * W, [&](long long first, long long count) {
    RowCodesArgs r = a;
    r.x = reinterpret_cast<const T*>(a.x) + first * a.xs;
    r.codes = a.codes + first * a.cs;
    r.scale = a.scale + first;
    if (fast) hipLaunchKernelGGL((row_codes_kernel<T, true, W>), dim3((unsigned)count), dim3(64 * W), 0, s, r);
    else hipLaunchKernelGGL((row_codes_kernel<T, false, W>), dim3((unsigned)count), dim3(64 * W), 0, s, r);
    return hipGetLastError();
  });
}
hipError_t launch_row_codes(const RowCodesArgs& a, bool bf16_in, hipStream_t s) {
  const bool wide = a.K > 64 * 8 * I8_KEEP;
  if (bf16_in) return wide ? codes_w<bf16, 4>(a, s) : codes_w<bf16, 1>(a, s);
  return wide ? codes_w<float, 4>(a, s) : codes_w<float, 1>(a, s);
}

template <typename T, int TM, int TN, int WM, int WN, int BUF> static hipError_t tile_t(const Int8LinearArgs& a, hipStream_t s) {
  auto kern = int8_tile_kernel<T, TM, TN, WM, WN, BUF>;
  const size_t lds = BUF * (TM + TN) * 128;
  const hipError_t e = set_lds_limit((const void*)kern, lds);
  if (e != hipSuccess) return e;
  const long long tiles = (long long)((a.M + TM - 1) / TM) * ((a.N + TN - 1) / TN);  // (below 2^23: int8_linear_fits)
  hipLaunchKernelGGL(kern, dim3((unsigned)tiles), dim3(64 * WM * WN), lds, s, a);
  return hipGetLastError();
}
template <typename T, int MT> static hipError_t few_t(Int8LinearArgs a, hipStream_t s) {
  return launch_slices((a.N + 15) / 16, 512, [&](long long first, long long count) {
    const dim3 grid((unsigned)count, (a.M + 16 * MT - 1) / (16 * MT));
    a.first = (int)first;
    hipLaunchKernelGGL((int8_few_kernel<T, MT, 0, false>), grid, dim3(512), 0, s, a);
    return hipGetLastError();
  });
}
template <typename T, int MT, int OWN> static hipError_t own_t(const Int8LinearArgs& a, hipStream_t s) {
  const bool fast = a.K % 8 == 0 && aligned16<T>(a.x, {a.xs});
  const size_t lds = (size_t)std::min(a.M, 16 * MT) * ((a.K + 127) / 128 * 128 + 16);
  const dim3 grid((a.N + 15) / 16, (a.M + 16 * MT - 1) / (16 * MT));
  if (fast) hipLaunchKernelGGL((int8_few_kernel<T, MT, OWN, true>), grid, dim3(512), lds, s, a);
  else hipLaunchKernelGGL((int8_few_kernel<T, MT, OWN, false>), grid, dim3(512), lds, s, a);
  return hipGetLastError();
}
template <typename T> static hipError_t linear_t(const Int8LinearArgs& a, int form, hipStream_t s) {
  switch (form) {
    case I8_OWN_8: return own_t<T, 1, 1>(a, s);
    case I8_OWN_16: return own_t<T, 1, 2>(a, s);
    case I8_OWN_32: return own_t<T, 2, 4>(a, s);
    case I8_FEW_16: return few_t<T, 1>(a, s);
    case I8_FEW_32: return few_t<T, 2>(a, s);
    case I8_TILE_64: return tile_t<T, 64, 64, 2, 2, 4>(a, s);
    case I8_TILE_128: return tile_t<T, 128, 128, 2, 2, 2>(a, s);
    default: return tile_t<T, 256, 256, 2, 4, 2>(a, s);
  }
}
hipError_t launch_int8_linear(const Int8LinearArgs& a, bool bf16_out, int form, hipStream_t s) {
  return bf16_out ? linear_t<bf16>(a, form, s) : linear_t<float>(a, form, s);
}

// Whether the largest tiles of a product fit one launch: y has at least 500 GB where they do not.
bool int8_linear_fits(int M, int N) { return ((M + 255ll) / 256) * ((N + 255ll) / 256) <= launch_most(512); }

// Which kernel a product takes.  Calls in a graph (us, M x K x N) that form the codes in the product's workgroups and that take a
// kernel for them: 1 x 4096 x 4096 5.6, 7.4; 8 x 4096 x 4096 8.2, 9.0; 8 x 2048 x 4096 6.2, 9.0; 16 x 2048 x 4096 8.0, 9.7;
// 16 x 512 x 512 6.1, 5.4; 32 x 1024 x 4096 7.7, 8.9; 300 x 1024 x 300 8.4, 9.5; 97 x 64 x 64 5.8, 5.4;
// 1 x 4096 x 11008 11.4, 12.5; 8 x 4096 x 11008 16.6, 15.6; 4 x 512 x 32768 20.6, 12.1.  fp32 tokens: 1 x 4096 x 4096 5.8, 7.5; 8 x 4096 x 4096 7.8, 8.5; 16 x
// 2048 x 4096 6.8, 8.7; 32 x 1024 x 4096 7.5, 8.5; 97 x 512 x 512 6.6, 6.3; 16 x 512 x 512 5.8, 5.4.  (A launch less saves 3 to
// 4 us of the caller's time besides: that is what decides where the kernels are even or a little behind.)
// Codes and product of 1 / 2 tiles of 16 tokens and of 64 x 64, 128 x 128 and 256 x 256 tiles:
//   M 16, K 4096, N 4096     10.1  10.3  12.3  25.0  50.4
//   32, 4096, 4096              -  11.9  12.5  25.4  50.5
//   64, 4096, 4096              -  17.4  12.8  25.9  50.5
//   97, 512, 512                -   6.4   6.8   9.7  13.8
//   200, 6000, 500              -  15.8  18.9  37.6  77.0
//   65, 6000, 6000              -  44.9  18.5  41.3  70.9
//   512, 4096, 4096             -  93.2  23.3  29.5  55.0
//   1024, 4096, 4096            -   179  41.4  34.7  56.9
//   2048, 4096, 4096            -   352  72.8  51.0  61.5
//   4096, 4096, 4096            -   694   128   102  81.9
// So: few tokens, or too few tiles to go round, the first; the largest tiles of which there is about one a CU.
int int8_linear_form(int M, int K, int N) {
  auto tiles = [&](int t) { return ((M + t - 1ll) / t) * ((N + t - 1ll) / t); };
  if (M <= 32 || tiles(64) < 48) {
    if (N <= I8_OWN_N && M <= 8 && K <= I8_OWN) return I8_OWN_8;
    if (N <= I8_OWN_N && M <= 16 && K <= I8_OWN / 2) return I8_OWN_16;
    if (N <= I8_OWN_N && M > 16 && K <= I8_OWN / 4) return I8_OWN_32;
    return M <= 16 ? I8_FEW_16 : I8_FEW_32;
  }
  return tiles(256) >= 224 ? I8_TILE_256 : tiles(128) >= 224 ? I8_TILE_128 : I8_TILE_64;
}

}  // namespace dfl
