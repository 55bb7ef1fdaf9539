// Rolling caches in 8 or 4 bits: prompts quantised as they are written, and caches (these and plain ones) read back in
// the order of their positions.
//
// A thread takes 8 elements of a row of the keys and the same of the values: 16 bytes of bf16 rows, 4 or 8 bytes of
// codes, neighbouring threads neighbouring elements, so that a group's maximum is two exchanges within a quad of lanes.
// A workgroup has whole rows (GR groups each: 64, 32, 21 or 16 of them), so that no thread divides a 64-bit index.
#include "launch_slices.h"
#include "lowbit_args.h"
#include "lowbit_codes.h"

#include <initializer_list>

namespace dfl {

// Bounds: memory.  135 MB of bf16 prompts into 4 bits (32 x 8 heads, 1028 slots, d 128), 170 MB in all: 44 us (3.9 TB/s)
// between readings of the caches, which leave nothing of the prompts in the last level of the caches; 35.5 in a row of fills
// of two batches in turn, of which that level holds a part (and workgroups of 128 slots that hand over whole lines of
// exponents, with two or four rows' loads in flight, 37).  What takes the time between readings is not settled: 8 bits, 204 MB,
// take 37 us, 5.5 TB/s.  fp32 prompts 57.5 and 62.6 us.  Reading back: 4 bits 29 us, 5.9 TB/s, 8 bits 37, 5.5, plain caches 44,
// 6.1.
template <int BITS> __device__ __forceinline__ void store_codes(const LowbitCache& q, int b, int hk, int s, int c,
                                                                const unsigned (&w)[BITS / 4], unsigned e) {
  uint8_t* to = q.codes + b * q.sb + hk * q.sh + s * q.sn + c * BITS;
  if constexpr (BITS == 4) *reinterpret_cast<unsigned*>(to) = w[0];
  else *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
  if (c % 4 == 0) q.exps[b * q.esb + hk * q.esh + c / 4 * q.esg + s] = (uint8_t)e;
}
template <typename T, int BITS, int GR, bool FAST> __global__ void __launch_bounds__(256) lowbit_fill_kernel(LowbitFillArgs a) {
  constexpr int NCH = 4 * GR, ROWS = 256 / NCH;
  const int S = a.n_sink + a.window;
  const int bh = blockIdx.y, b = bh / a.Hk, hk = bh % a.Hk;
  const int n = min(a.lengths[b], a.N), start = a.starts ? a.starts[b] : 0;
  if (n <= 0 || start < 0) return;
  const unsigned last = (unsigned)start + (unsigned)n - 1;  // at most 2^31 + 2^28
  // Latest position that a slot holds: past the first tokens, turn `turns` of the window up to the slot of `last`, one
  // turn less behind it.
  const unsigned past = last >= (unsigned)a.n_sink ? last - a.n_sink : 0u, turns = past / a.window;
  const unsigned rest = past - turns * a.window;
  const int s = (a.first + blockIdx.x) * ROWS + threadIdx.x / NCH, c = threadIdx.x % NCH;
  if ((int)threadIdx.x >= ROWS * NCH || s >= S || (unsigned)s > last) return;
  const unsigned o = (unsigned)(s - a.n_sink), back = o > rest;
  if (s >= a.n_sink && turns < back) return;
  const unsigned p = s < a.n_sink ? (unsigned)s : a.n_sink + o + (turns - back) * a.window;
  if (p < (unsigned)start) return;
  const size_t row = p - (unsigned)start;
  Eight<T> k, v;
  load8<FAST>(k, reinterpret_cast<const T*>(a.k) + b * a.ksb + hk * a.ksh + row * a.ksn, c, a.d);
  load8<FAST>(v, reinterpret_cast<const T*>(a.v) + b * a.vsb + hk * a.vsh + row * a.vsn, c, a.d);
  unsigned kw[BITS / 4], vw[BITS / 4];
  const unsigned ke = lb_encode<BITS>(k, kw), ve = lb_encode<BITS>(v, vw);
  store_codes<BITS>(a.kc, b, hk, s, c, kw, ke);
  store_codes<BITS>(a.vc, b, hk, s, c, vw, ve);
}

// BITS 0: a plain cache of T.
template <typename T, int BITS, bool FAST>
__device__ __forceinline__ void read_row(const LowbitCache& c, T* out, int b, int hk, int s, int ch, int d) {
  float x[8];
  if constexpr (BITS == 0) {
    const T* row = reinterpret_cast<const T*>(c.codes) + b * c.sb + hk * c.sh + s * c.sn;
    load8<T, FAST>(row, ch, d, x);
  } else {
    const uint8_t* at = c.codes + b * c.sb + hk * c.sh + s * c.sn + ch * BITS;
    unsigned w[BITS / 4];
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i) w[i] = reinterpret_cast<const unsigned*>(at)[i];
    lb_decode<BITS>(w, c.exps[b * c.esb + hk * c.esh + ch / 4 * c.esg + s], x);
  }
  store8<T, FAST>(out, ch, d, x);
}

template <typename T, int BITS, int GR, bool FAST> __global__ void __launch_bounds__(256) cache_read_kernel(CacheReadArgs a) {
  constexpr int NCH = 4 * GR, ROWS = 256 / NCH;
  const int S = a.n_sink + a.window;
  const int bh = blockIdx.y, b = bh / a.Hk, hk = bh % a.Hk;
  const int len = a.lengths[b];
  const int j = (a.first + blockIdx.x) * ROWS + threadIdx.x / NCH, c = threadIdx.x % NCH;
  if ((int)threadIdx.x >= ROWS * NCH || j >= S || c * 8 >= a.d) return;
  const int p = j < a.n_sink ? j : max(len, 0) - S + j;  // S < 2^29: no overflow
  const bool held = j < a.n_sink ? j < len : p >= a.n_sink;
  const size_t at = ((size_t)bh * S + j) * a.d;
  T* k = reinterpret_cast<T*>(a.k) + at;
  T* v = reinterpret_cast<T*>(a.v) + at;
  if (held) {
    const int s = p < a.n_sink ? p : a.n_sink + (p - a.n_sink) % a.window;
    read_row<T, BITS, FAST>(a.kc, k, b, hk, s, c, a.d);
    read_row<T, BITS, FAST>(a.vc, v, b, hk, s, c, a.d);
  } else {
    const float zero[8] = {};
    store8<T, FAST>(k, c, a.d, zero);
    store8<T, FAST>(v, c, a.d, zero);
  }
  if (hk == 0 && c == 0) a.mask[(size_t)b * S + j] = held ? 1.f : 0.f;
}

template <typename T> static bool aligned16(const void* p, std::initializer_list<long long> strides) {
  bool ok = ((uintptr_t)p & 15u) == 0;
  for (long long s : strides) ok = ok && ((s * (long long)sizeof(T)) & 15) == 0;
  return ok;
}

template <typename T, int BITS, int GR> static hipError_t fill_g(LowbitFillArgs a, hipStream_t s) {
  const bool fast = a.d % 8 == 0 && aligned16<T>(a.k, {a.ksb, a.ksh, a.ksn}) && aligned16<T>(a.v, {a.vsb, a.vsh, a.vsn});
  constexpr int ROWS = 256 / (4 * GR);
  return launch_slices((a.n_sink + a.window + ROWS - 1) / ROWS, 256, [&](long long first, long long count) {
    const dim3 grid((unsigned)count, a.B * a.Hk);
    a.first = (int)first;
    if (fast) hipLaunchKernelGGL((lowbit_fill_kernel<T, BITS, GR, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((lowbit_fill_kernel<T, BITS, GR, false>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
  });
}
template <typename T, int BITS> static hipError_t fill_b(const LowbitFillArgs& a, hipStream_t s) {
  switch (lb_groups(a.d)) {
    case 1: return fill_g<T, BITS, 1>(a, s);
    case 2: return fill_g<T, BITS, 2>(a, s);
    case 3: return fill_g<T, BITS, 3>(a, s);
    default: return fill_g<T, BITS, 4>(a, s);
  }
}
hipError_t launch_lowbit_fill(const LowbitFillArgs& a, bool bf16_in, int bits, hipStream_t s) {
  if (bf16_in) return bits == 4 ? fill_b<bf16, 4>(a, s) : fill_b<bf16, 8>(a, s);
  return bits == 4 ? fill_b<float, 4>(a, s) : fill_b<float, 8>(a, s);
}

template <typename T, int BITS, int GR> static hipError_t read_g(CacheReadArgs a, hipStream_t s) {
  bool fast = a.d % 8 == 0 && aligned16<T>(a.k, {}) && aligned16<T>(a.v, {});
  if (BITS == 0)
    fast = fast && aligned16<T>(a.kc.codes, {a.kc.sb, a.kc.sh, a.kc.sn}) && aligned16<T>(a.vc.codes, {a.vc.sb, a.vc.sh, a.vc.sn});
  constexpr int ROWS = 256 / (4 * GR);
  return launch_slices((a.n_sink + a.window + ROWS - 1) / ROWS, 256, [&](long long first, long long count) {
    const dim3 grid((unsigned)count, a.B * a.Hk);
    a.first = (int)first;
    if (fast) hipLaunchKernelGGL((cache_read_kernel<T, BITS, GR, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((cache_read_kernel<T, BITS, GR, false>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
  });
}
template <typename T, int BITS> static hipError_t read_b(const CacheReadArgs& a, hipStream_t s) {
  switch (lb_groups(a.d)) {
    case 1: return read_g<T, BITS, 1>(a, s);
    case 2: return read_g<T, BITS, 2>(a, s);
    case 3: return read_g<T, BITS, 3>(a, s);
    default: return read_g<T, BITS, 4>(a, s);
  }
}
template <typename T> static hipError_t read_t(const CacheReadArgs& a, int bits, hipStream_t s) {
  return bits == 4 ? read_b<T, 4>(a, s) : bits == 8 ? read_b<T, 8>(a, s) : read_b<T, 0>(a, s);
}
hipError_t launch_cache_read(const CacheReadArgs& a, bool bf16_out, int bits, hipStream_t s) {
  return bf16_out ? read_t<bf16>(a, bits, s) : read_t<float>(a, bits, s);
}

}  // namespace dfl
