// Learned bias by buckets of the relative position: out[b,h,i,j] = table[h, bucket(k_pos[j] - q_pos[i])], and the
// table's gradient, the sums of the bias's gradient over each bucket.
//
// Both directions only pass over the (M, N) planes, in flat 16-byte vectors (a plane's rows need no alignment).  The
// bucket comes from an LDS table over the distance, clipped to the largest edge.
#include "window_engine.h"

#include <algorithm>

namespace dfl {

// element vectors at any element alignment
template <typename T> struct Vec {
  static constexpr int N = 16 / (int)sizeof(T);
  T e[N];
};

struct RelPlane {
  const uint8_t* lut;
  const int *qp, *kp;  // the sample's positions, or null
  int N, shift, dist, lo;
  __device__ __forceinline__ RelPlane(const RelBiasArgs& a, const uint8_t* l, int b)
      : lut(l), qp(a.q_pos ? a.q_pos + (size_t)b * a.M : nullptr), kp(a.k_pos ? a.k_pos + (size_t)b * a.N : nullptr),
        N(a.N), shift(a.N - a.M), dist(a.rel.dist()), lo(a.rel.both ? a.rel.dist() : 0) {}
  // rel, clipped to the table of the LDS buckets; differences of two 32-bit positions take 33 bits
  __device__ __forceinline__ int bucket(int i, int j) const {
    const long long rel = qp ? (long long)kp[j] - qp[i] : (long long)j - i - shift;
    const int c = (int)min(max(rel, (long long)-dist), (long long)dist);
    return lut[lo ? c + lo : max(-c, 0)];
  }
};

// lut[c + dist] (one direction: lut[-c]) = bucket of rel = c, |c| <= dist
__device__ __forceinline__ void build_bucket_lut(const RelSpec& r, uint8_t* lut) {
  const int dist = r.dist(), n = r.both ? 2 * dist + 1 : dist + 1;
  for (int x = threadIdx.x; x < n; x += blockDim.x) lut[x] = (uint8_t)rel_bucket(r, r.both ? x - dist : -x);
}
static int bucket_lut_size(const RelSpec& r) { return ((r.both ? 2 * r.dist() + 1 : r.dist() + 1) + 15) & ~15; }

// A thread takes the buckets of one vector of the plane and writes it for every head.
template <typename T> __global__ void __launch_bounds__(256) rel_bias_fwd_kernel(RelBiasArgs a, int lut_bytes) {
  extern __shared__ __align__(16) unsigned char smem[];
  uint8_t* lut = smem;
  float* tab = reinterpret_cast<float*>(smem + lut_bytes);
  const int nb = a.rel.buckets(), b = blockIdx.y;
  const int h0 = blockIdx.z * 64, hn = min(64, a.H - h0);
  build_bucket_lut(a.rel, lut);
  for (int x = threadIdx.x; x < hn * nb; x += 256) tab[x] = a.table[(size_t)h0 * nb + x];
  __syncthreads();
  const RelPlane pl(a, lut, b);
  const size_t plane = (size_t)a.M * a.N, step = (size_t)gridDim.x * 256 * Vec<T>::N;
  for (size_t e0 = ((size_t)blockIdx.x * 256 + threadIdx.x) * Vec<T>::N; e0 < plane; e0 += step) {
    int i = (int)(e0 / a.N), j = (int)(e0 - (size_t)i * a.N), bk[Vec<T>::N];
    const int n = (int)min((size_t)Vec<T>::N, plane - e0);
#pragma unroll
    for (int v = 0; v < Vec<T>::N; ++v) {
      bk[v] = v < n ? pl.bucket(i, j) : 0;
      if (++j == a.N) j = 0, ++i;
    }
    T* out = reinterpret_cast<T*>(a.out) + ((size_t)b * a.H + h0) * plane + e0;
    for (int h = 0; h < hn; ++h, out += plane) {
      Vec<T> x;
#pragma unroll
      for (int v = 0; v < Vec<T>::N; ++v) x.e[v] = from_f32<T>(tab[h * nb + bk[v]]);
      if (n == Vec<T>::N) {
        __builtin_memcpy(out, &x, 16);
      } else {
        for (int v = 0; v < n; ++v) out[v] = x.e[v];
      }
    }
  }
}

// A workgroup sums its part of one plane by bucket: every thread has a column of its own in LDS, so no address has
// two writers and the order of each sum is fixed.
template <typename T> __global__ void __launch_bounds__(256) rel_bias_bwd_kernel(RelBiasArgs a, int lut_bytes) {
  extern __shared__ __align__(16) unsigned char smem[];
  uint8_t* lut = smem;
  float* hist = reinterpret_cast<float*>(smem + lut_bytes);
  const int nb = a.rel.buckets(), bh = blockIdx.y, b = bh / a.H;
  build_bucket_lut(a.rel, lut);
  for (int n = 0; n < nb; ++n) hist[n * 256 + threadIdx.x] = 0.f;
  __syncthreads();
  const RelPlane pl(a, lut, b);
  const size_t plane = (size_t)a.M * a.N, step = (size_t)gridDim.x * 256 * Vec<T>::N;
  const T* g = reinterpret_cast<const T*>(a.grad) + (size_t)bh * plane;
  for (size_t e0 = ((size_t)blockIdx.x * 256 + threadIdx.x) * Vec<T>::N; e0 < plane; e0 += step) {
    int i = (int)(e0 / a.N), j = (int)(e0 - (size_t)i * a.N);
    const int n = (int)min((size_t)Vec<T>::N, plane - e0);
    Vec<T> x;
    if (n == Vec<T>::N) {
      __builtin_memcpy(&x, g + e0, 16);
    } else {
      for (int v = 0; v < Vec<T>::N; ++v) x.e[v] = v < n ? g[e0 + v] : from_f32<T>(0.f);
    }
#pragma unroll
    for (int v = 0; v < Vec<T>::N; ++v) {
      if (v < n) hist[pl.bucket(i, j) * 256 + threadIdx.x] += to_f32(x.e[v]);
      if (++j == a.N) j = 0, ++i;
    }
  }
  __syncthreads();
  const int lane = threadIdx.x & 63;
  float* part = a.part + ((size_t)bh * a.n_part + blockIdx.x) * nb;
  for (int n = threadIdx.x >> 6; n < nb; n += 4) {
    const f32x4 s = *reinterpret_cast<const f32x4*>(hist + n * 256 + 4 * lane);
    const float t = wave_sum((s[0] + s[1]) + (s[2] + s[3]));
    if (lane == 0) part[n] = t;
  }
}

// dtable[h, n]: a wave for each
__global__ void __launch_bounds__(256) rel_bias_sum_kernel(RelBiasArgs a) {
  const int nb = a.rel.buckets(), w = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (w >= a.H * nb) return;
  const int h = w / nb, n = w % nb;
  float s = 0.f;
  for (int e = lane; e < a.B * a.n_part; e += 64)
    s += a.part[(((size_t)(e / a.n_part) * a.H + h) * a.n_part + e % a.n_part) * nb + n];
  s = wave_sum(s);
  if (lane == 0) a.dtable[w] = s;
}

hipError_t launch_rel_bias_fwd(const RelBiasArgs& a, bool bf16_out, hipStream_t s) {
  const int vec = bf16_out ? 8 : 4, lut = bucket_lut_size(a.rel);
  const size_t per = 256 * (size_t)vec, plane = (size_t)a.M * a.N;
  const unsigned nx = (unsigned)std::min<size_t>((plane + per - 1) / per, 2048);
  const size_t lds = lut + (size_t)std::min(a.H, 64) * a.rel.buckets() * 4;
  auto kern = bf16_out ? rel_bias_fwd_kernel<bf16> : rel_bias_fwd_kernel<float>;
  hipLaunchKernelGGL(kern, dim3(nx, a.B, (a.H + 63) / 64), dim3(256), lds, s, a, lut);
  return hipGetLastError();
}

int rel_bias_parts(int B, int H, int M, int N) {
  const size_t n = (size_t)M * N, want = std::max<size_t>(1, 2048 / ((size_t)B * H));
  return (int)std::max<size_t>(1, std::min<size_t>(want, (n + 2047) / 2048));
}

hipError_t launch_rel_bias_bwd(const RelBiasArgs& a, bool bf16_in, hipStream_t s) {
  const int lut = bucket_lut_size(a.rel), nb = a.rel.buckets();
  const size_t lds = lut + (size_t)nb * 1024;
  auto kern = bf16_in ? rel_bias_bwd_kernel<bf16> : rel_bias_bwd_kernel<float>;
  hipError_t e = set_lds_limit((const void*)kern, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3(a.n_part, a.B * a.H), dim3(256), lds, s, a, lut);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  hipLaunchKernelGGL(rel_bias_sum_kernel, dim3((a.H * nb + 3) / 4), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace dfl
