// Building blocks of the window attention kernels: 32x32 MFMA tiles over LDS tiles of
// 16-byte chunks.
//
// Every product is one of two kinds.
//  * row product: D[m][n] = sum_c A[m][c] R[n][c]; A rows from an LDS tile (one 16-byte chunk
//    a lane), R the wave's 32 resident rows, kept in registers (Frag).  bf16 takes
//    32x32x16 instructions (lane: row l % 32, columns 8 (l / 32) ..), fp32 four 32x32x2 a
//    chunk; both operands use the same column order, so any order gives the product.
//  * column product: O[c][n] += sum_m A[m][c] P[m][n] with P in the accumulator layout
//    (lane: n = l % 32, register r: m = 8 (r / 4) + 4 (l / 32) + r % 4).  As the B operand
//    the registers 8 s .. 8 s + 7 hold, in lane half h, the rows 16 s + 4 h + {0..3} and
//    16 s + 8 + 4 h + {0..3}; the A operand takes the same rows of the LDS tile
//    transposed, two ds_read_b64_tr_b16 (fp32: one 32-bit read a register).
// So scores are kept transposed (keys x queries) in the query-resident passes and queries x
// keys in the key-resident one: a softmax row never leaves its lane pair (l, l ^ 32), and
// probabilities go from accumulator to operand without passing through LDS.
//
// An LDS tile has rows of DP elements without padding; the 16-byte chunk c of row r lies at
// position c ^ f(r).  f sends 16 consecutive rows to 16 different positions of the 256-byte
// bank period (row reads of 16 bytes) and 4 consecutive rows to different 64-byte quarters
// (the transposing reads take 64 bytes of 4 rows at once), so neither read has conflicts.
#pragma once
#include "common.h"
#include "window_args.h"

#include <type_traits>

namespace dfl {

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;
typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4;
typedef __attribute__((__vector_size__(4 * sizeof(unsigned)))) unsigned u32x4;

constexpr int WIN_NT = 256;  // threads of a workgroup: 4 waves of 32 resident rows each
constexpr int WIN_RES = 128;

template <typename T, int DP> struct WinEng {
  static constexpr int VEC = 16 / (int)sizeof(T);  // elements of a chunk
  static constexpr int NCH = DP / VEC;             // chunks of a row
  static constexpr int STEPS = NCH / 2;            // chunk pairs: steps of a row product
  static constexpr int NT = DP / 32;               // 32-column tiles of a column product
  static constexpr int BK = (sizeof(T) == 4 && DP == 128) ? 32 : 64;  // streamed rows of an LDS tile
  static constexpr int NSUB = BK / 32;
  static constexpr int TILE = BK * DP;  // elements
  struct Frag { u32x4 v[STEPS]; };

  __device__ static __forceinline__ int swz(int r, int c) {
    if (NCH >= 16) return c ^ (((r & 3) << 2) | ((r >> 2) & 3));
    if (NCH == 8) return c ^ ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
    return c ^ ((r >> 2) & 3);
  }
  __device__ static __forceinline__ u32x4* chunk(T* tile, int r, int c) {
    return reinterpret_cast<u32x4*>(tile + r * DP + swz(r, c) * VEC);
  }

  // Chunk c of a global row (null: zeros); columns from d on are zero.  FAST: 16-byte
  // aligned rows and d a multiple of VEC.
  template <bool FAST> __device__ static __forceinline__ u32x4 load(const T* row, int c, int d) {
    u32x4 x = {0u, 0u, 0u, 0u};
    if (!row) return x;
    if (FAST) {
      if (c * VEC < d) x = *reinterpret_cast<const u32x4*>(row + c * VEC);
    } else {
      T e[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[i] = c * VEC + i < d ? row[c * VEC + i] : from_f32<T>(0.f);
      __builtin_memcpy(&x, e, 16);
    }
    return x;
  }
  // The wave's resident rows: lane l takes row l % 32 (its own `row`; null: zeros).
  template <bool FAST> __device__ static __forceinline__ void load_frag(Frag& f, const T* row, int d, int lane) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) f.v[s] = load<FAST>(row, 2 * s + (lane >> 5), d);
  }
  __device__ static __forceinline__ f32x16 step(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (sizeof(T) == 2) {
      bf16x8 x, y;
      __builtin_memcpy(&x, &a, 16);
      __builtin_memcpy(&y, &b, 16);
      c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    }
    return c;
  }
  // A lane's LDS addresses differ by one bit pattern a step (the swizzle is an exclusive or), so one register and
  // one instruction a read do.  `opaque` keeps them out of the loop-invariant set: the compiler would hold dozens of
  // them over the loop and spill, and a spilled register's reload waits for the tile loads in flight (key pass 180 ->
  // 150 us).  HELD: left to it, where there is room (forward 392 -> 372 us at 8192 tokens).
  __device__ static __forceinline__ unsigned opaque(unsigned x) {
    asm volatile("" : "+v"(x));
    return x;
  }
  __device__ static __forceinline__ unsigned lds_address(const T* p) {
    return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) T*)p;
  }
  // rows r0 .. r0 + 31 of the tile times the resident rows
  template <bool HELD = false>
  __device__ static __forceinline__ f32x16 row_product(T* tile, int r0, const Frag& f, int lane) {
    typedef const __attribute__((address_space(3))) u32x4* lptr;
    f32x16 c = {};
    const int row = lane & 31;  // (r0 a multiple of 32: the same swizzle)
    const unsigned base = lds_address(tile + r0 * DP);
    const unsigned own = row * DP * (unsigned)sizeof(T) + 16u * swz(row, lane >> 5), at = HELD ? own : opaque(own);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) c = step(*(lptr)(uintptr_t)(base + (at ^ (32u * s))), f.v[s], c);
    // a few LDS reads ahead of the products (the scheduler would rather save their registers and wait for each)
    constexpr int AHEAD = STEPS < 4 ? STEPS : 4, PER = sizeof(T) == 2 ? 1 : 4;
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
    for (int s = AHEAD; s < STEPS; ++s) {
      __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, AHEAD * PER, 0);
    return c;
  }
  // B operands of a column product
  typedef typename std::conditional<sizeof(T) == 2, bf16x8, f32x16>::type ProbV;
  struct Prob {
    ProbV h[sizeof(T) == 2 ? 2 : 1];
  };
  // bf16: probabilities and score gradients are rounded to bf16 here, as their products' other operand is;
  // the sums stay in fp32.  (A half step of 2^-8 each, of random sign: results are off by 0.0022-0.0024 of their size
  // where fp32 operands, at a sixteenth of the matrix rate, leave 0.0016-0.0017, the results' own rounding.)
  __device__ static __forceinline__ void to_operand(const f32x16& p, Prob& o) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int r = 0; r < 16; ++r) o.h[r / 8][r % 8] = (bf16)p[r];
    } else {
      o.h[0] = p;
    }
  }
  // s + the sum of a bf16 operand's values, as they were rounded
  __device__ static __forceinline__ float operand_sum(const Prob& p, float s) {
    typedef __attribute__((__vector_size__(2 * sizeof(bf16)))) bf16 pair;
    const pair ones = {(bf16)1.f, (bf16)1.f};
    pair x[8];
    __builtin_memcpy(x, &p, sizeof(x));
#pragma unroll
    for (int n = 0; n < 8; ++n) s = __builtin_amdgcn_fdot2_f32_bf16(x[n], ones, s, false);
    return s;
  }
  // acc[t] += (columns 32 t .. of rows r0 .. r0 + 31 of the tile)^T P
  template <bool HELD = false>
  __device__ static __forceinline__ void column_product(T* tile, int r0, const Prob& p, f32x16 (&acc)[NT], int lane) {
    if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) s16x4* lptr;
      const int h = lane >> 5, q = (lane >> 4) & 1, i = (lane & 15) >> 2, e = lane & 3, ra = 4 * h + i;
      constexpr unsigned RB = DP * 2;  // bytes of a row
      const unsigned base = lds_address(tile + r0 * DP);
      // 8 bytes of columns 16 q + 4 e .. of row 4 h + i; the row 8 further down has its chunks exchanged in pairs
      const unsigned own = ra * RB + 16u * swz(ra, 2 * q + (e >> 1)) + 8u * (e & 1), at = HELD ? own : opaque(own);
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)(uintptr_t)(base + 16 * s * RB + (at ^ (64u * t))));
          const s16x4 hi =
              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)(uintptr_t)(base + (16 * s + 8) * RB + (at ^ (64u * t + 32u))));
          bf16x8 a;
          __builtin_memcpy(&a, &lo, 8);
          __builtin_memcpy(reinterpret_cast<char*>(&a) + 8, &hi, 8);
          acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, p.h[s], acc[t], 0, 0, 0);
        }
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = r0 + 8 * (r / 4) + 4 * (lane >> 5) + r % 4;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int col = 32 * t + (lane & 31);
          const float a = tile[row * DP + swz(row, col / VEC) * VEC + col % VEC];
          acc[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p.h[0][r], acc[t], 0, 0, 0);
        }
      }
    }
  }
};

// Row of register r in lane half h of an accumulator tile.
__device__ __forceinline__ constexpr int acc_row(int r, int h) { return 8 * (r / 4) + 4 * h + r % 4; }

// Chunk-wise work order: workgroup w of n takes logical position x(w) such that each XCD (w mod 8) works on
// one contiguous part: neighbouring tiles, which read the same keys, share its L2.
__device__ __forceinline__ int xcd_order(int w, int n) {
  const int per = n >> 3, rem = n & 7, x = w & 7;
  return x * per + min(x, rem) + (w >> 3);
}

// ---------------------------------------------------------------------------
// Bias lookup in LDS: lut[x] for the distance x = t - j + base, in units of log2 (window_geometry.h).
constexpr int REL_EDGES = 96;  // ints of the edges in LDS, behind a lookup table
// bucket of rel = j - t
__device__ __forceinline__ int rel_bucket(const RelSpec& r, int rel) {
  const int mag = r.both ? abs(rel) : max(-rel, 0);
  int b = 0;
  for (int k = 0; k < r.n; ++k) b += r.edge[k] <= mag;
  return b + ((r.both && rel > 0) ? r.n + 1 : 0);
}
// The same from edges in LDS, by bisection.
__device__ __forceinline__ int rel_bucket_lds(const int* edge, int n, int both, int rel) {
  const int mag = both ? abs(rel) : max(-rel, 0);
  int b = 0;
#pragma unroll
  for (int step = 64; step; step >>= 1)
    if (b + step <= n && edge[b + step - 1] <= mag) b += step;
  return b + ((both && rel > 0) ? n + 1 : 0);
}
// Edges to LDS; the caller synchronises before they are read.
__device__ __forceinline__ void stage_edges(const RelSpec& r, int* edge) {
  if ((int)threadIdx.x < r.n) edge[threadIdx.x] = r.edge[threadIdx.x];
}
__device__ __forceinline__ void build_rel_lut(const WinArgs& a, int h, const int* edge, float* lut) {
  const int n = rel_lut_size(a.rel), base = rel_lut_base(a.rel);
  const float* row = a.table + (size_t)h * a.rel.buckets();
  for (int x = threadIdx.x; x < n; x += blockDim.x) {
    lut[x] = row[rel_bucket_lds(edge, a.rel.n, a.rel.both, base - x)] * LOG2E;
  }
}

}  // namespace dfl
