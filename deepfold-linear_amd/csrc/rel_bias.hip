// Learned bias by buckets of the relative position: out[b,h,i,j] = table[h, bucket(k_pos[j] - q_pos[i])], and the
// table's gradient, the sums of the bias's gradient over each bucket.
//
// Both directions only pass over the (M, N) planes, in flat 16-byte vectors (a plane's rows need no alignment).  The
// bucket comes from an LDS table over the distance, clipped to the largest edge.
//
// Bounds: the plane's bytes, once.  Forward 16 us for 34 MB (16 heads of 1024 x 1024 in bf16: half of it launch and the
// tables in LDS) and 58 us for 155 MB (4 x 16 of 777 x 777 in fp32, where a row's 16-byte stores start at any element);
// backward 17 and 94 us: a thread's read-add-write of its column for each run of one bucket, a chain of LDS latencies.
#include "window_engine.h"

#include <algorithm>

namespace dfl {

// element vectors at any element alignment
template <typename T> struct Vec {
  static constexpr int N = 16 / (int)sizeof(T);
  T e[N];
};

// Buckets of V consecutive elements of a sample's (M, N) plane from (i, j) on, over the rows' ends.
template <bool POS> struct RelPlane {
  const uint8_t* lut;
  const int *qp, *kp;  // the sample's positions
  int M, N, shift, dist, lo;
  __device__ __forceinline__ RelPlane(const RelBiasArgs& a, const uint8_t* l, int b)
      : lut(l), qp(POS ? a.q_pos + (size_t)b * a.M : nullptr), kp(POS ? a.k_pos + (size_t)b * a.N : nullptr), M(a.M),
        N(a.N), shift(a.N - a.M), dist(a.rel.dist()), lo(a.rel.both ? a.rel.dist() : 0) {}
  // a difference of two 32-bit positions saturates far outside the table
  __device__ __forceinline__ int bucket(int k, int q) const {
    const int c = min(max(__builtin_elementwise_sub_sat(k, q), -dist), dist);
    return lut[lo ? c + lo : max(-c, 0)];
  }
  template <int V> __device__ __forceinline__ void buckets(int i, int j, int (&bk)[V]) const {
    if (i >= M) {
#pragma unroll
      for (int v = 0; v < V; ++v) bk[v] = 0;
    } else if (j + V <= N) {
      int k[V];
      const int q = POS ? qp[i] : i + shift;
      if (POS) {
        __builtin_memcpy(k, kp + j, sizeof(k));
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) k[v] = j + v;
      }
#pragma unroll
      for (int v = 0; v < V; ++v) bk[v] = bucket(k[v], q);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        bk[v] = i < M ? bucket(POS ? kp[j] : j, POS ? qp[i] : i + shift) : bk[v ? v - 1 : 0];
        if (++j == N) j = 0, ++i;
      }
    }
  }
};
// Walks a plane in equal steps without a division a step.
struct PlaneWalk {
  int i, j, di, dj, N;
  __device__ __forceinline__ PlaneWalk(size_t first, size_t step, int n) : N(n) {
    if ((first | step) < (1ull << 32)) {  // 64-bit divisions take a microsecond
      i = (int)((unsigned)first / (unsigned)n);
      j = (int)((unsigned)first - (unsigned)i * n);
      di = (int)((unsigned)step / (unsigned)n);
      dj = (int)((unsigned)step - (unsigned)di * n);
      return;
    }
    i = (int)(first / n);
    j = (int)(first - (size_t)i * n);
    di = (int)(step / n);
    dj = (int)(step - (size_t)di * n);
  }
  __device__ __forceinline__ void next() {
    i += di;
    j += dj;
    if (j >= N) j -= N, ++i;
  }
};

// lut[c + dist] (one direction: lut[-c]) = bucket of rel = c, |c| <= dist; ends in a barrier
__device__ __forceinline__ void build_bucket_lut(const RelSpec& r, uint8_t* lut, int* edge) {
  const int dist = r.dist(), n = r.both ? 2 * dist + 1 : dist + 1;
  stage_edges(r, edge);
  __syncthreads();
  for (int x = threadIdx.x; x < n; x += blockDim.x)
    lut[x] = (uint8_t)rel_bucket_lds(edge, r.n, r.both, r.both ? x - dist : -x);
  __syncthreads();
}
static int bucket_lut_size(const RelSpec& r) { return ((r.both ? 2 * r.dist() + 1 : r.dist() + 1) + 15) & ~15; }

// A thread takes the buckets of one vector of the plane and writes it for every head.
template <typename T, bool POS>
__global__ void __launch_bounds__(256) rel_bias_fwd_kernel(RelBiasArgs a, int lut_bytes) {
  extern __shared__ __align__(16) unsigned char smem[];
  uint8_t* lut = smem;
  int* edge = reinterpret_cast<int*>(smem + lut_bytes);
  float* tab = reinterpret_cast<float*>(edge + REL_EDGES);
  const int nb = a.rel.buckets(), b = blockIdx.y;
  const int h0 = blockIdx.z * 64, hn = min(64, a.H - h0);
  for (int x = threadIdx.x; x < hn * nb; x += 256) tab[x] = a.table[(size_t)h0 * nb + x];
  build_bucket_lut(a.rel, lut, edge);
  const RelPlane<POS> pl(a, lut, b);
  const size_t plane = (size_t)a.M * a.N, step = (size_t)gridDim.x * 256 * Vec<T>::N;
  size_t e0 = ((size_t)blockIdx.x * 256 + threadIdx.x) * Vec<T>::N;
  PlaneWalk at(e0, step, a.N);
  for (; e0 < plane; e0 += step, at.next()) {
    int bk[Vec<T>::N];
    const int n = (int)min((size_t)Vec<T>::N, plane - e0);
    pl.buckets(at.i, at.j, bk);
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
// two writers and the order of each sum is fixed.  Neighbours of one bucket, most of them away from the diagonal, are
// added up before the column is touched; BWD_U vectors of a thread are loaded at once (one at a time, loads in flight
// bound the pass to a quarter of the memory rate).  A thread adds up at most BWD_CHAIN elements in fp32, whatever the
// plane's size (an error of at most BWD_CHAIN half steps of a column's sum of magnitudes); the parts are joined in 64
// bits.
constexpr int BWD_U = 4;
constexpr int BWD_CHAIN = 1024;
template <typename T, bool POS>
__global__ void __launch_bounds__(256) rel_bias_bwd_kernel(RelBiasArgs a, int lut_bytes) {
  constexpr int V = Vec<T>::N;
  extern __shared__ __align__(16) unsigned char smem[];
  uint8_t* lut = smem;
  int* edge = reinterpret_cast<int*>(smem + lut_bytes);
  float* hist = reinterpret_cast<float*>(edge + REL_EDGES);
  const int nb = a.rel.buckets(), bh = blockIdx.y, b = bh / a.H;
  for (int n = 0; n < nb; ++n) hist[n * 256 + threadIdx.x] = 0.f;
  build_bucket_lut(a.rel, lut, edge);
  const RelPlane<POS> pl(a, lut, b);
  const size_t plane = (size_t)a.M * a.N, row = 256 * (size_t)V, step = (size_t)gridDim.x * row;
  const T* g = reinterpret_cast<const T*>(a.grad) + (size_t)bh * plane;
  float* mine = hist + threadIdx.x;
  size_t e0 = (size_t)blockIdx.x * row + threadIdx.x * V;
  PlaneWalk at(e0, step, a.N);
  while (e0 < plane) {
    Vec<T> x[BWD_U];
    int bk[BWD_U][V];
#pragma unroll
    for (int u = 0; u < BWD_U; ++u) {
      const size_t e = e0 + u * step;
      if (e + V <= plane) {
        __builtin_memcpy(&x[u], g + e, 16);
      } else {  // (past the plane's end: zeros, into a bucket that is there)
#pragma unroll
        for (int v = 0; v < V; ++v) x[u].e[v] = e + v < plane ? g[e + v] : from_f32<T>(0.f);
      }
    }
#pragma unroll
    for (int u = 0; u < BWD_U; ++u) {
      pl.buckets(at.i, at.j, bk[u]);
      at.next();
    }
#pragma unroll
    for (int u = 0; u < BWD_U; ++u) {
      float s = to_f32(x[u].e[0]);
#pragma unroll
      for (int v = 1; v < V; ++v) {
        if (bk[u][v] != bk[u][v - 1]) {
          mine[bk[u][v - 1] * 256] += s;
          s = 0.f;
        }
        s += to_f32(x[u].e[v]);
      }
      mine[bk[u][V - 1] * 256] += s;
    }
    e0 += BWD_U * step;
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
  double s = 0.;
  for (int e = lane; e < a.B * a.n_part; e += 64)
    s += a.part[(((size_t)(e / a.n_part) * a.H + h) * a.n_part + e % a.n_part) * nb + n];
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, WAVE);
  if (lane == 0) a.dtable[w] = (float)s;
}

hipError_t launch_rel_bias_fwd(const RelBiasArgs& a, bool bf16_out, hipStream_t s) {
  const int vec = bf16_out ? 8 : 4, lut = bucket_lut_size(a.rel);
  const size_t per = 256 * (size_t)vec, plane = (size_t)a.M * a.N;
  // at most about 4 workgroups a CU in all: each builds its lookup table once
  const unsigned nx = (unsigned)std::min<size_t>((plane + per - 1) / per, std::max(1, 1024 / a.B));
  const size_t lds = lut + REL_EDGES * 4 + (size_t)std::min(a.H, 64) * a.rel.buckets() * 4;
  auto kern = a.q_pos ? (bf16_out ? rel_bias_fwd_kernel<bf16, true> : rel_bias_fwd_kernel<float, true>)
                      : (bf16_out ? rel_bias_fwd_kernel<bf16, false> : rel_bias_fwd_kernel<float, false>);
  hipLaunchKernelGGL(kern, dim3(nx, a.B, (a.H + 63) / 64), dim3(256), lds, s, a, lut);
  return hipGetLastError();
}

// Parts of a plane: about 4 workgroups a CU in all, at least one round of vectors each, at most BWD_CHAIN elements a
// thread (the last vector of a thread's share may be one more; 2^20 parts are planes beyond any memory).
int rel_bias_parts(int B, int H, int M, int N) {
  const size_t n = (size_t)M * N, want = std::max<size_t>(1, 1024 / ((size_t)B * H));
  const size_t chains = n > 256 * BWD_CHAIN ? n / (256 * (BWD_CHAIN - 8)) + 1 : 1;
  return (int)std::min<size_t>(1 << 20, std::max(chains, std::min<size_t>(want, (n + 4095) / 4096)));
}

hipError_t launch_rel_bias_bwd(const RelBiasArgs& a, bool bf16_in, hipStream_t s) {
  const int lut = bucket_lut_size(a.rel), nb = a.rel.buckets();
  const size_t lds = lut + REL_EDGES * 4 + (size_t)nb * 1024;
  auto kern = a.q_pos ? (bf16_in ? rel_bias_bwd_kernel<bf16, true> : rel_bias_bwd_kernel<float, true>)
                      : (bf16_in ? rel_bias_bwd_kernel<bf16, false> : rel_bias_bwd_kernel<float, false>);
  hipError_t e = set_lds_limit((const void*)kern, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3(a.n_part, a.B * a.H), dim3(256), lds, s, a, lut);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  hipLaunchKernelGGL(rel_bias_sum_kernel, dim3((a.H * nb + 3) / 4), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace dfl
