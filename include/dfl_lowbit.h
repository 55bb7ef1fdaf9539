/*
 * Parameter blocks of the operators of a layer served in few bits, declared in dfl_amd.h
 * (dfl_lowbit_*, dfl_window_cache_read, dfl_quantize_rows, dfl_int8_linear): rolling caches held
 * in 8 or 4 bits, one token's attention over them, and products in 8-bit integers.
 * Conventions as in dfl_amd.h and dfl_window.h.
 *
 * Codes: 32 elements of a row form a group, the last one filled up with zeros.  A group's
 * exponent byte E stands for 2^(E - 127); an element's value is its code times that.
 *   8 bits: an integer in [-127, 127], two's complement.
 *   4 bits: bit 3 the sign, bits 2..0 one of 0, 0.5, 1, 1.5, 2, 3, 4, 6; the even element
 *           in a byte's low half.
 * E is the lowest, from 1 on, with which the group's largest magnitude is below 127.5 * 2^(E - 127) (8 bits)
 * or at most 7 * 2^(E - 127) (4 bits), so that no element is off by more than half a step; E of groups that reach 2^127
 * is at most 248 or 252, which keeps all values finite, and their largest elements take the last code.
 * Codes are the nearest, ties to the even one.  A group that holds an infinity or NaN has E =
 * 255 and codes 0, and reads as NaN.
 */
#ifndef DFL_LOWBIT_H
#define DFL_LOWBIT_H

/* A rolling cache of S = n_sink + window slots: codes (B,Hk,S,G * 4 * bits bytes), G = ceil(d / 32) groups,
 * and exponent bytes (B,Hk,G,S'), a group's slots side by side, S' a multiple of 4 from S on (the bytes
 * behind the last slot may be read, never used).  Strides in bytes: the codes' and their pointer multiples of 16,
 * the exponents' of 4.  The decode takes row strides below 2^26 and group strides of at most 2^28 + 192 bytes. */
typedef struct dfl_lowbit_cache {
  void* codes;
  void* exponents;
  long long stride_b, stride_h, stride_n;
  long long exp_stride_b, exp_stride_h, exp_stride_g;
} dfl_lowbit_cache;

/* As dfl_window_cache_fill, into such caches: row i of k, v (B,Hk,N,d) stands at position
 * starts[b] + i (starts NULL: i), rows 0 .. lengths[b] - 1 count.  starts[b] < 0 leaves the sample's caches alone. */
typedef struct dfl_lowbit_cache_fill_params {
  int dtype, bits;
  const void* k;
  const void* v;
  long long k_stride_b, k_stride_h, k_stride_n;
  long long v_stride_b, v_stride_h, v_stride_n;
  const int* lengths;
  const int* starts;
  dfl_lowbit_cache k_cache, v_cache;
  int B, Hk, N, d, window, n_sink;
} dfl_lowbit_cache_fill_params;

/* A cache's rows in the order of their positions: k, v (B,Hk,S,d) contiguous in `dtype`, of row j < n_sink position j, of
 * any other lengths[b] - S + j, where lengths[b] positions have entered; mask (B,S) fp32: 1 where the row has such a
 * position (j < lengths[b]; n_sink <= lengths[b] - S + j), else 0 and the row zero.  bits 4 or 8: such caches; bits 0:
 * codes points to elements in `dtype`, strides in elements, exponents unused. */
typedef struct dfl_window_cache_read_params {
  int dtype, bits;
  dfl_lowbit_cache k_cache, v_cache;
  const int* lengths;
  void* k;
  void* v;
  float* mask;
  int B, Hk, d, window, n_sink;
} dfl_window_cache_read_params;

/* As dfl_window_decode, over such caches: the token's own key and value enter them, and count, as their codes stand.
 * A sample and key head with a group of E = 255 among its slots in use: zero divided by zero in every output.  Values up to
 * the largest that a group holds are weighted without passing fp32 on the way (weights below 2^-88 of the largest may
 * vanish beside such values, else those below 2^-125). */
typedef struct dfl_lowbit_decode_params {
  int dtype, bits;
  const void* q;
  const void* k;
  const void* v;
  long long q_stride_b, q_stride_h;
  long long k_stride_b, k_stride_h;
  long long v_stride_b, v_stride_h;
  dfl_lowbit_cache k_cache, v_cache;
  const int* lengths;
  const float* rel_table;
  const int* rel_edges;
  int n_edges;
  int B, H, Hk, d, window, n_sink;
  float scale;
  void* o;
} dfl_lowbit_decode_params;

/* Rows x (M,K), row stride x_stride, as codes (M,K) int8 with row stride code_stride >= K (a multiple of 16, as the
 * pointer is; the bytes from K on are written as zeros) and scale (M) fp32: scale = max(max |x| / 127 rounded to fp32,
 * 2^-100), code the integer nearest to x / scale, ties to even.  A row that holds an infinity or NaN has scale NaN and
 * codes 0. */
typedef struct dfl_quantize_rows_params {
  int dtype;
  const void* x;
  long long x_stride;
  long long M;
  int K;
  void* codes;
  long long code_stride;
  float* scale;
} dfl_quantize_rows_params;

/* y (M,N) contiguous in `dtype`: y[m,n] = (sum_k a[m,k] w[n,k]) s[m] w_scale[n] + bias[n] with a, s the codes and
 * scale of x's rows as in dfl_quantize_rows and w (N,K) int8 codes; bias in `dtype` or NULL.  The sum is exact (K at
 * most 131072; M and N at most 2^31 - 256, and ceil(M / 256) ceil(N / 256) below 2^23).  w and its row stride (bytes) are
 * multiples of 16, and a row's bytes up to the next multiple of 16 from K on are read, whatever they hold. */
typedef struct dfl_int8_linear_params {
  int dtype;
  const void* x;
  long long x_stride;
  const void* w;
  long long w_stride;
  const float* w_scale;
  const void* bias;
  void* y;
  int M, K, N;
} dfl_int8_linear_params;

#endif
