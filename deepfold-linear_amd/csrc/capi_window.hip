// C-ABI entry points of the sequence operators (include/dfl_window.h): argument checks, work split, workspace
// layout and launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "../../include/dfl_amd.h"
#include "window_args.h"

namespace dfl {
int capi_fail(const char* message);
int capi_hip_fail(hipError_t e, const char* what);
hipError_t launch_window_fwd(const WinArgs& a, bool bf16_in, int DP, hipStream_t s);
hipError_t launch_window_bwd(const WinArgs& a, bool bf16_in, int DP, hipStream_t s);
hipError_t launch_cache_fill(const CacheFillArgs& a, bool bf16_in, hipStream_t s);
hipError_t launch_window_decode(const DecodeArgs& a, bool bf16_in, int DP, hipStream_t s);
hipError_t launch_rel_bias_fwd(const RelBiasArgs& a, bool bf16_out, hipStream_t s);
hipError_t launch_rel_bias_bwd(const RelBiasArgs& a, bool bf16_in, hipStream_t s);
int rel_bias_parts(int B, int H, int M, int N);
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

constexpr int RES = 128;          // resident rows of a workgroup (window_engine.h: WIN_RES)
constexpr long long MAX_N = 1ll << 28;  // positions and their differences stay well inside 32 bits
constexpr int MAX_SINK = 128;

int pad_dim(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }
size_t r256(size_t n) { return (n + 255) / 256 * 256; }

bool edges_ok(int n, int both) { return n >= 0 && n <= (both ? (dfl::REL_MAX_EDGES + 1) / 2 - 1 : dfl::REL_MAX_EDGES); }
int check_rel(const int* edges, int n, int both) {
  if (n < 0 || (n > 0 && !edges)) return fail("rel_edges is NULL");
  if (!edges_ok(n, both))
    return fail("%d edges give more than %d buckets", n, dfl::REL_MAX_EDGES + 1);
  for (int i = 0; i < n; ++i) {
    if (edges[i] < 1 || edges[i] > dfl::REL_MAX_DIST) return fail("edge %d outside [1, %d]", edges[i], dfl::REL_MAX_DIST);
    if (i && edges[i] <= edges[i - 1]) return fail("rel_edges must ascend");
  }
  return 0;
}
dfl::RelSpec rel_spec(const int* edges, int n, int both) {
  dfl::RelSpec r;
  memset(&r, 0, sizeof(r));
  r.n = n;
  r.both = both;
  for (int i = 0; i < n; ++i) r.edge[i] = edges[i];
  return r;
}
// A product of two ints fits 64 bits: tested first, so that none of the sizes formed from it can wrap around.
constexpr long long MAX_BH = 1ll << 22;  // four waves for each of 128 first tokens of each are counted in 32 bits
bool heads_ok(int B, int H, int Hk, int d) {
  return B > 0 && H > 0 && Hk > 0 && H % Hk == 0 && d > 0 && d <= 128 && (long long)B * H < MAX_BH;
}
bool window_ok(int window, int n_sink) { return window >= 1 && n_sink >= 0 && n_sink <= MAX_SINK; }

int check_heads(int dtype, int B, int H, int Hk, int d) {
  if (dtype != DFL_F32 && dtype != DFL_BF16) return fail("dtype must be DFL_F32 or DFL_BF16");
  if (B <= 0 || H <= 0 || Hk <= 0) return fail("B, H, Hk must be positive");
  if (H % Hk != 0) return fail("H=%d is no multiple of Hk=%d", H, Hk);
  if (d <= 0 || d > 128) return fail("head dim d=%d outside [1, 128]", d);
  if (!heads_ok(B, H, Hk, d)) return fail("B * H = %lld is too large", (long long)B * H);
  return 0;
}
// The running reference is a maximum of scaled scores, taken before the scale.
int check_scale(float scale) {
  return scale >= 1e-30f && scale <= 1e30f ? 0 : fail("scale=%g outside [1e-30, 1e30]", (double)scale);
}
int check_window(int window, int n_sink) {
  if (window < 1) return fail("window=%d must be positive", window);
  if (n_sink < 0 || n_sink > MAX_SINK) return fail("n_sink=%d outside [0, %d]", n_sink, MAX_SINK);
  return 0;
}

// Query chunks of the first tokens' gradients: about 32 a (sample, key head), of whole tiles; none where every
// query's band reaches every first token.
struct Chunks {
  int n, size;
  Chunks(int M, int N, int window, int n_sink, int causal) : n(0), size(0) {
    if (n_sink == 0 || N <= window) return;
    const int first = causal ? std::max(0, window - (N - M)) : 0, rows = M - first;
    if (rows <= 0) return;
    size = std::max(256, (rows + 31) / 32);
    size = (size + RES - 1) / RES * RES;
    n = (rows + size - 1) / size;
  }
};

// Parts of a key tile's queries (window_attn_bwd.hip: 64 keys, 64 queries a step).  Below two workgroups a CU the
// key pass waits for its own loads and barriers most of the time: at 16 / 4 heads of 4096 tokens, 256 workgroups,
// window 1024, it takes 171 us in one part and, with 10 us more for joining them, 146 us in two; four gave the same as
// two.  A part has at least 8 steps, so that the joining stays small beside it.  Whole training steps (us) in one part,
// by this rule, and with twice the workgroups and half the steps: 16 / 4 heads of 4096 tokens, d 128 as above 294, 270,
// 275; 8 of 2048, d 64, window 512 68, 68, 77; 2 x 8 / 2 of 1500, d 64, 200 both ways 115, 83, 87; fp32 8 / 2 of 2000,
// d 64, window 700 467, 266, 272; 32 / 8 of 1024, d 128 216, 134, 139; 4 / 1 of 600, d 64, all both ways 118, 66, 60;
// fp32 4 of 1000, d 32, 300 both ways 146, 146, 131; fp32 8 of 4096, d 128, window 1024 844, 840, 885.
int kv_split(int B, int H, int Hk, int M, int N, int window, int causal) {
  const long long tiles = ((long long)N + 63) / 64 * B * Hk;
  const long long w = std::min(window, N), band = std::min<long long>(M, 63 + (causal ? w : 2 * w - 1));
  const long long steps = (long long)(H / Hk) * ((band + 63) / 64);
  int s = 1;
  while (s < 8 && tiles * s < 512 && steps / (2 * s) >= 8) s *= 2;
  return s;
}

struct WindowWs {
  size_t rowd, sink, kv, tab, total;
  WindowWs(int B, int H, int Hk, int M, int N, int d, int window, int n_sink, int causal, int n_edges) {
    const Chunks c(M, N, window, n_sink, causal);
    const size_t DP = pad_dim(d), nqt = ((size_t)M + RES - 1) / RES, nb = causal ? n_edges + 1 : 2 * (n_edges + 1);
    rowd = 0;
    sink = r256((size_t)B * H * M * 8);
    kv = sink + r256(c.n ? (size_t)B * Hk * (c.n + 1) * std::min(n_sink, N) * 2 * DP * 4 : 0);
    const int split = kv_split(B, H, Hk, M, N, window, causal);
    tab = kv + r256(split > 1 ? (size_t)split * B * Hk * N * 2 * DP * 4 : 0);
    total = tab + r256(n_edges > 0 ? (size_t)B * H * nqt * nb * 4 : 0);
  }
};

int check_attn(const dfl_window_attn_params* p, bool bwd) {
  if (!p) return fail("params is NULL");
  if (int rc = check_heads(p->dtype, p->B, p->H, p->Hk, p->d)) return rc;
  if (int rc = check_window(p->window, p->n_sink)) return rc;
  if (p->M <= 0 || p->N <= 0 || p->M > p->N || p->N > MAX_N)
    return fail("M=%d, N=%d: need 0 < M <= N <= %lld", p->M, p->N, MAX_N);
  if ((((long long)p->N + 63) / 64 + 1) * p->B * p->H * 8 >= (1ll << 31)) return fail("too many rows");
  if (int rc = check_scale(p->scale)) return rc;
  if (!p->q || !p->k || !p->v || !p->o) return fail("required pointer is NULL");
  if (!p->rel_table != (p->n_edges == 0)) return fail("rel_table and rel_edges must be given together");
  if (int rc = check_rel(p->rel_edges, p->n_edges, !p->causal)) return rc;
  if (bwd && (!p->lse || !p->grad_o || !p->dq || !p->dk || !p->dv)) return fail("gradient pointer is NULL");
  if (bwd && p->drel_table && !p->rel_table) return fail("drel_table without rel_table");
  return 0;
}

dfl::WinArgs attn_args(const dfl_window_attn_params* p) {
  dfl::WinArgs a;
  memset(&a, 0, sizeof(a));
  a.q = p->q; a.k = p->k; a.v = p->v;
  a.qsb = p->q_stride_b; a.qsh = p->q_stride_h; a.qsn = p->q_stride_n;
  a.ksb = p->k_stride_b; a.ksh = p->k_stride_h; a.ksn = p->k_stride_n;
  a.vsb = p->v_stride_b; a.vsh = p->v_stride_h; a.vsn = p->v_stride_n;
  a.mask = p->mask;
  a.table = p->rel_table;
  a.rel = rel_spec(p->rel_edges, p->n_edges, !p->causal);
  a.B = p->B; a.H = p->H; a.Hk = p->Hk; a.M = p->M; a.N = p->N; a.d = p->d;
  a.window = p->window; a.n_sink = p->n_sink; a.causal = p->causal != 0;
  a.scale = p->scale;
  a.o = p->o;
  a.o_rest = p->o_rest;
  a.lse = p->lse;
  return a;
}

// Splits of a cache: about three workgroups a CU, what the registers of the bf16 form with four heads a group let run at
// once (with 1024 a second, mostly empty round follows), at least 64 slots each.  Calls (us) with 512, 768 and 1024:
// bf16 32 x 32 / 8 heads, 4100 slots, d 128 125, 117, 132; fp32 8 x 32 / 8, the same 52, 54, 55; bf16 16 x 16, 2052
// slots, d 64 31, 31, 31; fp32 8 x 16, 504 slots, d 32, table 17, 16, 17; bf16 1 x 16 / 4, 1028 slots, d 64 20, 15, 20;
// 1 x 32 / 8, 16388 slots, d 128 30, 30, 35.
constexpr int DECODE_WG = 768, DECODE_MIN = 64;
struct Splits {
  int n, chunk;
  Splits(int B, int H, int Hk, int S) {
    const long long wg = (long long)B * Hk * ((H / Hk + 3) / 4);
    const long long want = std::max<long long>(1, DECODE_WG / wg), most = (S + DECODE_MIN - 1) / DECODE_MIN;
    n = (int)std::min(want, most);
    chunk = (S + n - 1) / n;
    n = (S + chunk - 1) / chunk;
  }
};

int check_bias(const dfl_rel_bias_params* p) {
  if (!p) return fail("params is NULL");
  if (p->dtype != DFL_F32 && p->dtype != DFL_BF16) return fail("dtype must be DFL_F32 or DFL_BF16");
  if (p->B <= 0 || p->H <= 0 || p->M <= 0 || p->N <= 0 || p->M > MAX_N || p->N > MAX_N)
    return fail("B, H, M, N must be positive and M, N at most %lld", MAX_N);
  if ((long long)p->B * p->H > 65535) return fail("B * H = %lld > 65535", (long long)p->B * p->H);
  if ((long long)p->B * dfl::rel_bias_parts(p->B, p->H, p->M, p->N) >= (1ll << 31)) return fail("M * N is too large");
  if (!p->q_pos != !p->k_pos) return fail("q_pos and k_pos must be given together");
  if (p->n_edges < 1) return fail("rel_edges is empty");
  return check_rel(p->rel_edges, p->n_edges, p->rel_both);
}
dfl::RelBiasArgs bias_args(const dfl_rel_bias_params* p) {
  dfl::RelBiasArgs a;
  memset(&a, 0, sizeof(a));
  a.table = p->rel_table;
  a.rel = rel_spec(p->rel_edges, p->n_edges, p->rel_both != 0);
  a.q_pos = p->q_pos; a.k_pos = p->k_pos;
  a.B = p->B; a.H = p->H; a.M = p->M; a.N = p->N;
  a.out = p->out;
  a.grad = p->grad_out;
  a.dtable = p->drel_table;
  return a;
}

}  // namespace

extern "C" {

size_t dfl_window_attn_workspace_size(int B, int H, int Hk, int M, int N, int d, int window, int n_sink, int causal,
                                      int n_edges) {
  if (!heads_ok(B, H, Hk, d) || M <= 0 || N < M || N > MAX_N || !window_ok(window, n_sink) || !edges_ok(n_edges, !causal))
    return 0;
  return WindowWs(B, H, Hk, M, N, d, window, n_sink, causal, n_edges).total;
}

int dfl_window_attn_fwd(const dfl_window_attn_params* p, void* stream) {
  return guarded([&] {
    if (int rc = check_attn(p, false)) return rc;
    const hipError_t e =
        dfl::launch_window_fwd(attn_args(p), p->dtype == DFL_BF16, pad_dim(p->d), (hipStream_t)stream);
    return e == hipSuccess ? 0 : dfl::capi_hip_fail(e, "window attention forward launch");
  });
}

int dfl_window_attn_bwd(const dfl_window_attn_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    if (int rc = check_attn(p, true)) return rc;
    const WindowWs w(p->B, p->H, p->Hk, p->M, p->N, p->d, p->window, p->n_sink, p->causal, p->n_edges);
    if (!workspace || workspace_bytes < w.total) return fail("workspace too small: need %zu bytes", w.total);
    dfl::WinArgs a = attn_args(p);
    const Chunks c(p->M, p->N, p->window, p->n_sink, p->causal);
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    a.go = p->grad_o;
    a.dq = p->dq; a.dk = p->dk; a.dv = p->dv;
    a.dtable = p->drel_table;
    a.rowd = reinterpret_cast<float*>(ws + w.rowd);
    a.sink_part = reinterpret_cast<float*>(ws + w.sink);
    a.tab_part = reinterpret_cast<float*>(ws + w.tab);
    a.kv_part = reinterpret_cast<float*>(ws + w.kv);
    a.kv_split = kv_split(p->B, p->H, p->Hk, p->M, p->N, p->window, p->causal);
    a.n_chunks = c.n;
    a.chunk = c.size;
    const hipError_t e = dfl::launch_window_bwd(a, p->dtype == DFL_BF16, pad_dim(p->d), (hipStream_t)stream);
    return e == hipSuccess ? 0 : dfl::capi_hip_fail(e, "window attention backward launch");
  });
}

int dfl_window_cache_append(const dfl_window_cache_fill_params* p, const int* starts, void* stream) {
  return guarded([&] {
    if (!p) return fail("params is NULL");
    if (int rc = check_heads(p->dtype, p->B, p->Hk, p->Hk, p->d)) return rc;
    if (int rc = check_window(p->window, p->n_sink)) return rc;
    if (p->N <= 0 || p->N > MAX_N || p->window > MAX_N) return fail("N and window must be in [1, %lld]", MAX_N);
    if ((long long)p->B * p->Hk > 65535) return fail("B * Hk = %lld > 65535", (long long)p->B * p->Hk);
    if (!p->k || !p->v || !p->lengths || !p->k_cache || !p->v_cache) return fail("required pointer is NULL");
    dfl::CacheFillArgs a;
    a.k = p->k; a.v = p->v;
    a.ksb = p->k_stride_b; a.ksh = p->k_stride_h; a.ksn = p->k_stride_n;
    a.vsb = p->v_stride_b; a.vsh = p->v_stride_h; a.vsn = p->v_stride_n;
    a.lengths = p->lengths;
    a.starts = starts;
    a.first = 0;
    a.kc = p->k_cache; a.vc = p->v_cache;
    a.kcsb = p->kc_stride_b; a.kcsh = p->kc_stride_h; a.kcsn = p->kc_stride_n;
    a.vcsb = p->vc_stride_b; a.vcsh = p->vc_stride_h; a.vcsn = p->vc_stride_n;
    a.B = p->B; a.Hk = p->Hk; a.N = p->N; a.d = p->d; a.window = p->window; a.n_sink = p->n_sink;
    const hipError_t e = dfl::launch_cache_fill(a, p->dtype == DFL_BF16, (hipStream_t)stream);
    return e == hipSuccess ? 0 : dfl::capi_hip_fail(e, "cache fill launch");
  });
}

int dfl_window_cache_fill(const dfl_window_cache_fill_params* p, void* stream) {
  return dfl_window_cache_append(p, nullptr, stream);
}

size_t dfl_window_decode_workspace_size(int B, int H, int Hk, int d, int window, int n_sink) {
  if (!heads_ok(B, H, Hk, d) || !window_ok(window, n_sink) || window > MAX_N) return 0;
  const Splits s(B, H, Hk, window + n_sink);
  return s.n > 1 ? r256((size_t)B * H * s.n * (pad_dim(d) + 2) * 4) : 0;
}

int dfl_window_decode(const dfl_window_decode_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    if (!p) return fail("params is NULL");
    if (int rc = check_heads(p->dtype, p->B, p->H, p->Hk, p->d)) return rc;
    if (int rc = check_window(p->window, p->n_sink)) return rc;
    if (p->window > MAX_N) return fail("window=%d above %lld", p->window, MAX_N);
    if (int rc = check_scale(p->scale)) return rc;
    if (!p->q || !p->k || !p->v || !p->k_cache || !p->v_cache || !p->lengths || !p->o)
      return fail("required pointer is NULL");
    if (!p->rel_table != (p->n_edges == 0)) return fail("rel_table and rel_edges must be given together");
    if (int rc = check_rel(p->rel_edges, p->n_edges, 0)) return rc;
    const size_t need = dfl_window_decode_workspace_size(p->B, p->H, p->Hk, p->d, p->window, p->n_sink);
    if (need && (!workspace || workspace_bytes < need)) return fail("workspace too small: need %zu bytes", need);
    dfl::DecodeArgs a;
    memset(&a, 0, sizeof(a));
    a.q = p->q; a.k = p->k; a.v = p->v;
    a.qsb = p->q_stride_b; a.qsh = p->q_stride_h; a.ksb = p->k_stride_b; a.ksh = p->k_stride_h;
    a.vsb = p->v_stride_b; a.vsh = p->v_stride_h;
    a.kc = p->k_cache; a.vc = p->v_cache;
    a.kcsb = p->kc_stride_b; a.kcsh = p->kc_stride_h; a.kcsn = p->kc_stride_n;
    a.vcsb = p->vc_stride_b; a.vcsh = p->vc_stride_h; a.vcsn = p->vc_stride_n;
    a.lengths = p->lengths;
    a.table = p->rel_table;
    a.rel = rel_spec(p->rel_edges, p->n_edges, 0);
    a.B = p->B; a.H = p->H; a.Hk = p->Hk; a.d = p->d; a.window = p->window; a.n_sink = p->n_sink;
    a.scale = p->scale;
    a.o = p->o;
    a.part = static_cast<float*>(workspace);
    const Splits s(p->B, p->H, p->Hk, p->window + p->n_sink);
    a.n_split = s.n;
    a.chunk = s.chunk;
    if ((long long)p->B * p->Hk * ((p->H / p->Hk + 3) / 4) * s.n >= (1ll << 31)) return fail("too many rows");
    const hipError_t e = dfl::launch_window_decode(a, p->dtype == DFL_BF16, pad_dim(p->d), (hipStream_t)stream);
    return e == hipSuccess ? 0 : dfl::capi_hip_fail(e, "window decode launch");
  });
}

size_t dfl_rel_bias_workspace_size(int B, int H, int M, int N, int n_edges, int rel_both) {
  if (B <= 0 || H <= 0 || M <= 0 || N <= 0 || M > MAX_N || N > MAX_N || (long long)B * H > 65535 || !edges_ok(n_edges, rel_both))
    return 0;
  return r256((size_t)B * H * dfl::rel_bias_parts(B, H, M, N) * (rel_both ? 2 : 1) * (n_edges + 1) * 4);
}

int dfl_rel_bias_fwd(const dfl_rel_bias_params* p, void* stream) {
  return guarded([&] {
    if (int rc = check_bias(p)) return rc;
    if (!p->rel_table || !p->out) return fail("required pointer is NULL");
    const hipError_t e = dfl::launch_rel_bias_fwd(bias_args(p), p->dtype == DFL_BF16, (hipStream_t)stream);
    return e == hipSuccess ? 0 : dfl::capi_hip_fail(e, "relative bias launch");
  });
}

int dfl_rel_bias_bwd(const dfl_rel_bias_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    if (int rc = check_bias(p)) return rc;
    if (!p->grad_out || !p->drel_table) return fail("gradient pointer is NULL");
    const size_t need = dfl_rel_bias_workspace_size(p->B, p->H, p->M, p->N, p->n_edges, p->rel_both);
    if (!workspace || workspace_bytes < need) return fail("workspace too small: need %zu bytes", need);
    dfl::RelBiasArgs a = bias_args(p);
    a.part = static_cast<float*>(workspace);
    a.n_part = dfl::rel_bias_parts(p->B, p->H, p->M, p->N);
    const hipError_t e = dfl::launch_rel_bias_bwd(a, p->dtype == DFL_BF16, (hipStream_t)stream);
    return e == hipSuccess ? 0 : dfl::capi_hip_fail(e, "relative bias backward launch");
  });
}

}  // extern "C"
