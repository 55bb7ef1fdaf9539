/*
 * Parameter blocks of the sequence operators declared in dfl_amd.h (dfl_window_*,
 * dfl_rel_bias_*): attention over a sliding window and a few first tokens, its
 * rolling cache and single-token form, and the learned bias by buckets of the
 * relative position.  Conventions as in dfl_amd.h; strides are in elements, with a
 * unit stride of the last dimension, and may be any value (0 included on inputs).
 *
 * Buckets: rel = key position - query position.  mag = |rel| with rel_both = 1, else
 * max(-rel, 0); bucket = number of edges <= mag, plus n_edges + 1 where rel_both = 1
 * and rel > 0.  rel_edges is a HOST array of n_edges ascending integers in
 * [1, 2048], read during the call; a table has n_edges + 1 buckets a head, or
 * 2 (n_edges + 1) with rel_both = 1, and at most 96.  n_edges = 0 with a NULL table:
 * no bias.
 */
#ifndef DFL_WINDOW_H
#define DFL_WINDOW_H

/* Queries (B,H,M,d), keys and values (B,Hk,N,d), H a multiple of Hk (query head h reads
 * key head h / (H / Hk)), M <= N: query i stands at position t = i + N - M.  It sees key j if
 * t - window < j <= t (causal = 0: |t - j| < window) or j < n_sink (causal: and j <= t),
 * and mask[b,j] != 0; rows with mask[b,t] = 0, or that see nothing, are zero.  The table's
 * direction is that of the attention: rel_both = !causal.  A table entry of -inf
 * (or below about -1e30) takes its keys out.  scale is positive (1e-30 to 1e30).
 *
 * Training: the forward writes lse (B,H,M) and, in bf16, o_rest (B,H,M,d), what the rounding of o leaves; both go to the
 * backward with o.  o_rest may be NULL: the backward then takes a pass more.  It is not read, nor written, where
 * dtype is fp32 or the rows see at most 256 keys. */
typedef struct dfl_window_attn_params {
  int dtype;
  const void* q;
  const void* k;
  const void* v;
  long long q_stride_b, q_stride_h, q_stride_n;
  long long k_stride_b, k_stride_h, k_stride_n;
  long long v_stride_b, v_stride_h, v_stride_n;
  const float* mask;
  const float* rel_table;
  const int* rel_edges;
  int n_edges;
  int B, H, Hk, M, N, d;
  int window, n_sink, causal;
  float scale;
  void* o;
  float* lse;
  const void* grad_o;
  void* dq;
  void* dk;
  void* dv;
  float* drel_table;
  void* o_rest;
} dfl_window_attn_params;

/* Rolling cache of S = n_sink + window slots (B,Hk,S,d): position p < n_sink lies in slot p,
 * any other in slot n_sink + (p - n_sink) % window.  Rows 0 .. lengths[b] - 1 of k, v (B,Hk,N,d)
 * go where they belong (the last one of those that share a slot); slots without a position
 * keep what they hold.  lengths (B) int32 on the device; above N counts as N. */
typedef struct dfl_window_cache_fill_params {
  int dtype;
  const void* k;
  const void* v;
  long long k_stride_b, k_stride_h, k_stride_n;
  long long v_stride_b, v_stride_h, v_stride_n;
  const int* lengths;
  void* k_cache;
  void* v_cache;
  long long kc_stride_b, kc_stride_h, kc_stride_n;
  long long vc_stride_b, vc_stride_h, vc_stride_n;
  int B, Hk, N, d, window, n_sink;
} dfl_window_cache_fill_params;

/* One token a sample: q (B,H,d), its key and value k, v (B,Hk,d) at position lengths[b].  The
 * key and value enter the cache; o (B,H,d) is the attention over the slots then in use.
 * lengths[b] < 0: zero output, cache row untouched.  The table's direction is one (rel_both = 0). */
typedef struct dfl_window_decode_params {
  int dtype;
  const void* q;
  const void* k;
  const void* v;
  long long q_stride_b, q_stride_h;
  long long k_stride_b, k_stride_h;
  long long v_stride_b, v_stride_h;
  void* k_cache;
  void* v_cache;
  long long kc_stride_b, kc_stride_h, kc_stride_n;
  long long vc_stride_b, vc_stride_h, vc_stride_n;
  const int* lengths;
  const float* rel_table;
  const int* rel_edges;
  int n_edges;
  int B, H, Hk, d, window, n_sink;
  float scale;
  void* o;
} dfl_window_decode_params;

/* out[b,h,i,j] = rel_table[h, bucket(k_pos[b,j] - q_pos[b,i])] in the element type `dtype`, (B,H,M,N)
 * contiguous; q_pos (B,M) and k_pos (B,N) int32, or both NULL: positions i + N - M and j.  Backward:
 * grad_out (B,H,M,N) contiguous in `dtype`, drel_table (H, buckets) fp32. */
typedef struct dfl_rel_bias_params {
  int dtype;
  const float* rel_table;
  const int* rel_edges;
  int n_edges, rel_both;
  const int* q_pos;
  const int* k_pos;
  int B, H, M, N;
  void* out;
  const void* grad_out;
  float* drel_table;
} dfl_rel_bias_params;

#endif
