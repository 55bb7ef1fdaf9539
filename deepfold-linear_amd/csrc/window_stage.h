// Staging of the window attention's tiles into LDS.
#pragma once
#include "window_engine.h"

namespace dfl {

// One 16-byte load a lane from `from` to `to` + 16 lane in LDS (`to` uniform, in bytes), not waited for: lds_loads_done().
// Written out because the compiler, where it knows of such a load, waits for all of them before the next transposing LDS
// read, whatever that reads; what it does not know of cannot make its own waits too short, since loads return in order.
__device__ __forceinline__ void load_to_lds(const void* from, unsigned to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(to) : "memory", "m0");
}
__device__ __forceinline__ void lds_loads_done() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0) alone; the builtin, so that the compiler knows its own loads done too
  asm volatile("" ::: "memory");
}

// Brings tiles of BK rows of one operand to LDS.  FAST: asynchronous 16-byte loads straight into LDS (no registers
// between, in flight until lds_loads_done() and a barrier); the swizzle is on the global side, each lane fetching the
// chunk that belongs where its 16 bytes land.  Rows from N on repeat the last one and chunks from column d on the
// row's first, so that every address is inside: clear_rows() zeroes such rows before use, and columns from d on meet
// zero columns of the resident operand or end in columns that are not written.  Else: element loads, zeros outside.
template <typename T, int DP, bool FAST> struct RowLoader {
  using E = WinEng<T, DP>;
  static constexpr int PER = E::BK * E::NCH / WIN_NT;  // chunks of a thread
  static constexpr int STEP = WIN_NT / E::NCH;         // rows between them
  long long stride, mine;  // mine: this thread's chunk of the rows from 0 on, in elements
  int N, d;
  __device__ __forceinline__ static int column(int row, int pos, int d) {
    const int c = E::swz(row, pos) * E::VEC;
    return c < d ? c : 0;
  }
  __device__ __forceinline__ RowLoader(long long s, int n, int dim) : stride(s), N(n), d(dim) {
    const int r = threadIdx.x / E::NCH;
    mine = r * stride + column(r, threadIdx.x % E::NCH, d);
  }
  __device__ __forceinline__ void issue(const T* base, T* tile, int j0) const {
    const int r = threadIdx.x / E::NCH, pos = threadIdx.x % E::NCH;
    if constexpr (FAST) {
      const unsigned to = __builtin_amdgcn_readfirstlane(E::lds_address(tile + (threadIdx.x & ~63u) * E::VEC));
      if (STEP % 16 == 0 && j0 + E::BK <= N) {  // one column for all of the thread's rows
        const T* from = base + j0 * stride + mine;
#pragma unroll
        for (int n = 0; n < PER; ++n, from += STEP * stride) load_to_lds(from, to + n * WIN_NT * 16);
      } else {
#pragma unroll
        for (int n = 0; n < PER; ++n) {
          const int row = r + n * STEP;
          load_to_lds(base + min(j0 + row, N - 1) * stride + column(row, pos, d), to + n * WIN_NT * 16);
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < PER; ++n) {
        const int row = r + n * STEP, j = j0 + row;
        *E::chunk(tile, row, pos) = E::template load<false>(j < N ? base + j * stride : nullptr, pos, d);
      }
    }
  }
};

// Zeroes the rows of a staged tile whose bit is clear: outside the sequence or masked, where NaN may lie.
template <typename T, int DP> __device__ __forceinline__ void clear_rows(T* tile, uint64_t bits) {
  using E = WinEng<T, DP>;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  for (int e = threadIdx.x; e < E::BK * E::NCH; e += WIN_NT)
    if (!((bits >> (e / E::NCH)) & 1u)) *reinterpret_cast<u32x4*>(tile + e * E::VEC) = zero;
}

// One bit for each of the BK rows from j0 on: inside [0, N) and unmasked; the same in every wave.  fetch() loads the
// mask ahead of its use, get() forms the bits.
template <int BK> struct RowBits {
  static constexpr uint64_t ALL = BK == 64 ? ~0ull : (1ull << BK) - 1;
  const float* mask;
  int N, at;
  float v;
  __device__ __forceinline__ RowBits(const float* m, int n) : mask(m), N(n), at(0), v(1.f) {}
  __device__ __forceinline__ void fetch(int j0) {
    at = j0;
    if (mask) v = mask[min(j0 + (int)(threadIdx.x & 63u), N - 1)];
  }
  __device__ __forceinline__ uint64_t get() const {
    if (!mask && at + BK <= N) return ALL;
    const int lane = threadIdx.x & 63;
    return __ballot((lane < BK) & (at + lane < N) & (v != 0.f));
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
