// C-ABI entry points of the operators of a layer served in few bits (include/dfl_lowbit.h): argument checks, work split,
// workspace layout and launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "../../include/dfl_amd.h"
#include "lowbit_args.h"

namespace dfl {
int capi_fail(const char* message);
int capi_hip_fail(hipError_t e, const char* what);
hipError_t launch_lowbit_fill(const LowbitFillArgs& a, bool bf16_in, int bits, hipStream_t s);
hipError_t launch_cache_read(const CacheReadArgs& a, bool bf16_out, int bits, hipStream_t s);
hipError_t launch_lowbit_decode(const LowbitDecodeArgs& a, bool bf16_in, int bits, int DP, hipStream_t s);
LowbitPlan lowbit_decode_plan(bool bf16_in, int B, int H, int Hk, int d, int S);
hipError_t launch_row_codes(const RowCodesArgs& a, bool bf16_in, hipStream_t s);
int int8_linear_form(int M, int K, int N);
bool int8_linear_fits(int M, int N);
hipError_t launch_int8_linear(const Int8LinearArgs& a, bool bf16_out, int form, hipStream_t s);
}  // namespace dfl

namespace {

int fail(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
int fail(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return dfl::capi_fail(buf);
}

// No exception leaves a C entry.
template <class F> int guarded(F f) {
  try {
    return f();
  } catch (...) {
    return fail("out of host memory");
  }
}

constexpr long long MAX_N = 1ll << 28;   // positions and their differences stay well inside 32 bits
constexpr long long MAX_BH = 1ll << 22;
constexpr int MAX_SINK = 128, MAX_K = 1 << 17;  // 2^17 products of two codes: below 2^31
constexpr int MAX_ROWS = 0x7fffff00;  // tokens, rows of weights: a tile that begins below it ends below 2^31

int pad_dim(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }
size_t r256(size_t n) { return (n + 255) / 256 * 256; }

// A product of two ints fits 64 bits: tested first, so that none of the sizes formed from it can wrap around.
bool heads_ok(int B, int H, int Hk, int d) {
  return B > 0 && H > 0 && Hk > 0 && H % Hk == 0 && d > 0 && d <= 128 && (long long)B * H < MAX_BH;
}
bool window_ok(int window, int n_sink) { return window >= 1 && window <= MAX_N && n_sink >= 0 && n_sink <= MAX_SINK; }

int check_shape(int dtype, int B, int H, int Hk, int d, int window, int n_sink) {
  if (dtype != DFL_F32 && dtype != DFL_BF16) return fail("dtype must be DFL_F32 or DFL_BF16");
  if (B <= 0 || H <= 0 || Hk <= 0) return fail("B, H, Hk must be positive");
  if (H % Hk != 0) return fail("H=%d is no multiple of Hk=%d", H, Hk);
  if (d <= 0 || d > 128) return fail("head dim d=%d outside [1, 128]", d);
  if (!heads_ok(B, H, Hk, d)) return fail("B * H = %lld is too large", (long long)B * H);
  if (window < 1 || window > MAX_N) return fail("window=%d outside [1, %lld]", window, MAX_N);
  if (n_sink < 0 || n_sink > MAX_SINK) return fail("n_sink=%d outside [0, %d]", n_sink, MAX_SINK);
  return 0;
}
// (Strides of dimensions of one element are not looked at.)
int check_codes(const dfl_lowbit_cache& c, int bits, int B, int Hk, int S, int d) {
  if (bits != 4 && bits != 8) return fail("bits must be 4 or 8");
  if (!c.codes || !c.exponents) return fail("required pointer is NULL");
  const uintptr_t codes = (uintptr_t)c.codes | (uintptr_t)(B > 1 ? c.stride_b : 0) | (uintptr_t)(Hk > 1 ? c.stride_h : 0) |
                          (uintptr_t)(S > 1 ? c.stride_n : 0);
  const uintptr_t exps = (uintptr_t)c.exponents | (uintptr_t)(B > 1 ? c.exp_stride_b : 0) |
                         (uintptr_t)(Hk > 1 ? c.exp_stride_h : 0) | (uintptr_t)(d > 32 ? c.exp_stride_g : 0);
  if (codes & 15) return fail("a cache's codes and their strides must be multiples of 16 bytes");
  if (exps & 3) return fail("a cache's exponents and their strides must be multiples of 4 bytes");
  return 0;
}
// The decode's offsets: 32 rows of codes, and a head's exponents, within 2^31 bytes; rows behind each other.
int check_near(const dfl_lowbit_cache& c, int bits, int d, int S) {
  const int groups = (d + 31) / 32;
  if (S > 1 && (c.stride_n < groups * 4 * bits || c.stride_n >= (1 << 26)))
    return fail("a cache's row stride must hold a row and be below 2^26 bytes");
  if (groups > 1 && (c.exp_stride_g < S || c.exp_stride_g > MAX_N + MAX_SINK + 64))
    return fail("a cache's group stride must hold the slots and be at most %lld bytes", MAX_N + MAX_SINK + 64);
  return 0;
}
dfl::LowbitCache cache(const dfl_lowbit_cache& c) {
  return {static_cast<uint8_t*>(c.codes), static_cast<uint8_t*>(c.exponents), c.stride_b, c.stride_h, c.stride_n,
          c.exp_stride_b, c.exp_stride_h, c.exp_stride_g};
}

size_t code_row(int K) { return ((size_t)K + 127) / 128 * 128; }
bool linear_ok(int M, int K, int N) { return M > 0 && K > 0 && N > 0 && K <= MAX_K; }
struct LinearWs {
  size_t scale, total;
  LinearWs(int M, int K) {
    scale = r256((size_t)M * code_row(K));
    total = scale + r256((size_t)M * 4);
  }
};

}  // namespace

extern "C" {

int dfl_lowbit_cache_fill(const dfl_lowbit_cache_fill_params* p, void* stream) {
  return guarded([&] {
    if (!p) return fail("params is NULL");
    if (int rc = check_shape(p->dtype, p->B, p->Hk, p->Hk, p->d, p->window, p->n_sink)) return rc;
    if (int rc = check_codes(p->k_cache, p->bits, p->B, p->Hk, p->window + p->n_sink, p->d)) return rc;
    if (int rc = check_codes(p->v_cache, p->bits, p->B, p->Hk, p->window + p->n_sink, p->d)) return rc;
    if (p->N <= 0 || p->N > MAX_N) return fail("N must be in [1, %lld]", MAX_N);
    if ((long long)p->B * p->Hk > 65535) return fail("B * Hk = %lld > 65535", (long long)p->B * p->Hk);
    if (!p->k || !p->v || !p->lengths) return fail("required pointer is NULL");
    dfl::LowbitFillArgs a;
    a.k = p->k; a.v = p->v;
    a.ksb = p->k_stride_b; a.ksh = p->k_stride_h; a.ksn = p->k_stride_n;
    a.vsb = p->v_stride_b; a.vsh = p->v_stride_h; a.vsn = p->v_stride_n;
    a.lengths = p->lengths; a.starts = p->starts;
    a.kc = cache(p->k_cache); a.vc = cache(p->v_cache);
    a.B = p->B; a.Hk = p->Hk; a.N = p->N; a.d = p->d; a.window = p->window; a.n_sink = p->n_sink;
    a.first = 0;
    const hipError_t e = dfl::launch_lowbit_fill(a, p->dtype == DFL_BF16, p->bits, (hipStream_t)stream);
    return e == hipSuccess ? 0 : dfl::capi_hip_fail(e, "few-bit cache fill launch");
  });
}

int dfl_window_cache_read(const dfl_window_cache_read_params* p, void* stream) {
  return guarded([&] {
    if (!p) return fail("params is NULL");
    if (int rc = check_shape(p->dtype, p->B, p->Hk, p->Hk, p->d, p->window, p->n_sink)) return rc;
    if (p->bits) {
      if (int rc = check_codes(p->k_cache, p->bits, p->B, p->Hk, p->window + p->n_sink, p->d)) return rc;
      if (int rc = check_codes(p->v_cache, p->bits, p->B, p->Hk, p->window + p->n_sink, p->d)) return rc;
    }
    if ((long long)p->B * p->Hk > 65535) return fail("B * Hk = %lld > 65535", (long long)p->B * p->Hk);
    if (!p->k_cache.codes || !p->v_cache.codes || !p->lengths || !p->k || !p->v || !p->mask)
      return fail("required pointer is NULL");
    dfl::CacheReadArgs a;
    a.kc = cache(p->k_cache); a.vc = cache(p->v_cache);
    a.lengths = p->lengths;
    a.k = p->k; a.v = p->v; a.mask = p->mask;
    a.B = p->B; a.Hk = p->Hk; a.d = p->d; a.window = p->window; a.n_sink = p->n_sink;
    a.first = 0;
    const hipError_t e = dfl::launch_cache_read(a, p->dtype == DFL_BF16, p->bits, (hipStream_t)stream);
    return e == hipSuccess ? 0 : dfl::capi_hip_fail(e, "cache read launch");
  });
}

size_t dfl_lowbit_decode_workspace_size(int B, int H, int Hk, int d, int window, int n_sink) {
  if (!heads_ok(B, H, Hk, d) || !window_ok(window, n_sink)) return 0;
  const int n = std::max(dfl::lowbit_decode_plan(true, B, H, Hk, d, window + n_sink).n_split,
                         dfl::lowbit_decode_plan(false, B, H, Hk, d, window + n_sink).n_split);
  return n > 1 ? r256((size_t)B * H * n * (pad_dim(d) + 2) * 4) : 0;
}

int dfl_lowbit_decode(const dfl_lowbit_decode_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    if (!p) return fail("params is NULL");
    if (int rc = check_shape(p->dtype, p->B, p->H, p->Hk, p->d, p->window, p->n_sink)) return rc;
    if (int rc = check_codes(p->k_cache, p->bits, p->B, p->Hk, p->window + p->n_sink, p->d)) return rc;
    if (int rc = check_codes(p->v_cache, p->bits, p->B, p->Hk, p->window + p->n_sink, p->d)) return rc;
    const int S = p->window + p->n_sink;
    if (int rc = check_near(p->k_cache, p->bits, p->d, S)) return rc;
    if (int rc = check_near(p->v_cache, p->bits, p->d, S)) return rc;
    if (!(p->scale >= 1e-30f && p->scale <= 1e30f)) return fail("scale=%g outside [1e-30, 1e30]", (double)p->scale);
    if (!p->q || !p->k || !p->v || !p->lengths || !p->o) return fail("required pointer is NULL");
    if (!p->rel_table != (p->n_edges == 0)) return fail("rel_table and rel_edges must be given together");
    if (p->n_edges < 0 || p->n_edges > dfl::REL_MAX_EDGES || (p->n_edges > 0 && !p->rel_edges))
      return fail("%d edges: need 0 to %d, and their array", p->n_edges, dfl::REL_MAX_EDGES);
    for (int i = 0; i < p->n_edges; ++i)
      if (p->rel_edges[i] < (i ? p->rel_edges[i - 1] + 1 : 1) || p->rel_edges[i] > dfl::REL_MAX_DIST)
        return fail("rel_edges must ascend within [1, %d]", dfl::REL_MAX_DIST);
    const size_t need = dfl_lowbit_decode_workspace_size(p->B, p->H, p->Hk, p->d, p->window, p->n_sink);
    if (need && (!workspace || workspace_bytes < need)) return fail("workspace too small: need %zu bytes", need);
    dfl::LowbitDecodeArgs a;
    memset(&a, 0, sizeof(a));
    a.q = p->q; a.k = p->k; a.v = p->v;
    a.qsb = p->q_stride_b; a.qsh = p->q_stride_h; a.ksb = p->k_stride_b; a.ksh = p->k_stride_h;
    a.vsb = p->v_stride_b; a.vsh = p->v_stride_h;
    a.kc = cache(p->k_cache); a.vc = cache(p->v_cache);
    if (S == 1) a.kc.sn = a.vc.sn = (p->d + 31) / 32 * 4 * p->bits;  // (of one row, any stride)
    a.lengths = p->lengths;
    a.table = p->rel_table;
    a.rel.n = p->n_edges;
    for (int i = 0; i < p->n_edges; ++i) a.rel.edge[i] = p->rel_edges[i];
    a.B = p->B; a.H = p->H; a.Hk = p->Hk; a.d = p->d; a.window = p->window; a.n_sink = p->n_sink;
    a.scale = p->scale;
    a.o = p->o;
    a.part = static_cast<float*>(workspace);
    const dfl::LowbitPlan plan = dfl::lowbit_decode_plan(p->dtype == DFL_BF16, p->B, p->H, p->Hk, p->d, S);
    a.waves = plan.waves;
    a.n_split = plan.n_split;
    a.chunk = plan.chunk;
    const int G = p->H / p->Hk;
    if ((long long)p->B * p->Hk * ((G + plan.heads - 1) / plan.heads) * plan.n_split >= (1ll << 31)) return fail("too many rows");
    const hipError_t e = dfl::launch_lowbit_decode(a, p->dtype == DFL_BF16, p->bits, pad_dim(p->d), (hipStream_t)stream);
    return e == hipSuccess ? 0 : dfl::capi_hip_fail(e, "few-bit decode launch");
  });
}

int dfl_quantize_rows(const dfl_quantize_rows_params* p, void* stream) {
  return guarded([&] {
    if (!p) return fail("params is NULL");
    if (p->dtype != DFL_F32 && p->dtype != DFL_BF16) return fail("dtype must be DFL_F32 or DFL_BF16");
    if (p->M <= 0 || p->M >= (1ll << 31) || p->K <= 0 || p->K > MAX_K)
      return fail("M=%lld, K=%d: need 0 < M < 2^31, 0 < K <= %d", p->M, p->K, MAX_K);
    if (!p->x || !p->codes || !p->scale) return fail("required pointer is NULL");
    if (p->code_stride < p->K || ((uintptr_t)p->codes | (uintptr_t)p->code_stride) & 15)
      return fail("codes and code_stride must be multiples of 16 bytes, code_stride at least K");
    const dfl::RowCodesArgs a = {p->x, p->x_stride, static_cast<int8_t*>(p->codes), p->code_stride, p->scale, p->M, p->K};
    const hipError_t e = dfl::launch_row_codes(a, p->dtype == DFL_BF16, (hipStream_t)stream);
    return e == hipSuccess ? 0 : dfl::capi_hip_fail(e, "row quantisation launch");
  });
}

size_t dfl_int8_linear_workspace_size(int M, int K, int N) {
  return linear_ok(M, K, N) && dfl::int8_linear_form(M, K, N) > dfl::I8_OWN_32 ? LinearWs(M, K).total : 0;
}

int dfl_int8_linear(const dfl_int8_linear_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    if (!p) return fail("params is NULL");
    if (p->dtype != DFL_F32 && p->dtype != DFL_BF16) return fail("dtype must be DFL_F32 or DFL_BF16");
    if (!linear_ok(p->M, p->K, p->N)) return fail("M=%d, K=%d, N=%d: need positive sizes and K <= %d", p->M, p->K, p->N, MAX_K);
    if (!p->x || !p->w || !p->w_scale || !p->y) return fail("required pointer is NULL");
    if (p->w_stride < p->K || ((uintptr_t)p->w | (uintptr_t)p->w_stride) & 15)
      return fail("w and w_stride must be multiples of 16 bytes, w_stride at least K");
    if (p->M > MAX_ROWS || p->N > MAX_ROWS) return fail("M=%d, N=%d: at most %d", p->M, p->N, MAX_ROWS);
    const int form = dfl::int8_linear_form(p->M, p->K, p->N);
    if (!dfl::int8_linear_fits(p->M, p->N)) return fail("M * N is too large");
    dfl::Int8LinearArgs a = {p->x, p->x_stride, nullptr, nullptr, static_cast<const int8_t*>(p->w), p->w_scale, p->bias, p->y,
                             0, p->w_stride, p->M, p->K, p->N, 0};
    hipError_t e;
    if (form > dfl::I8_OWN_32) {
      const LinearWs ws(p->M, p->K);
      if (!workspace || workspace_bytes < ws.total) return fail("workspace too small: need %zu bytes", ws.total);
      if ((uintptr_t)workspace & 15) return fail("workspace must be 16-byte aligned");
      unsigned char* at = static_cast<unsigned char*>(workspace);
      const dfl::RowCodesArgs r = {p->x, p->x_stride, reinterpret_cast<int8_t*>(at), (long long)code_row(p->K),
                                   reinterpret_cast<float*>(at + ws.scale), p->M, p->K};
      e = dfl::launch_row_codes(r, p->dtype == DFL_BF16, (hipStream_t)stream);
      if (e != hipSuccess) return dfl::capi_hip_fail(e, "row quantisation launch");
      a.a = r.codes;
      a.a_scale = r.scale;
      a.as = r.cs;
    }
    e = dfl::launch_int8_linear(a, p->dtype == DFL_BF16, form, (hipStream_t)stream);
    return e == hipSuccess ? 0 : dfl::capi_hip_fail(e, "8-bit product launch");
  });
}

}  // extern "C"
