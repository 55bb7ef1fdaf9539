// Argument blocks of the operators of a layer served in few bits (rolling caches in 8 or 4 bits, products in 8-bit
// integers), shared by the kernels and the C-ABI layer.  Semantics: include/dfl_lowbit.h.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "window_geometry.h"

namespace dfl {

struct LowbitCache {
  uint8_t* codes;     // (B,Hk,S,row bytes), byte strides, multiples of 16
  uint8_t* exps;      // (B,Hk,groups,S'), byte strides, multiples of 4
  long long sb, sh, sn;
  long long esb, esh, esg;
};

struct LowbitFillArgs {
  const void* k;  // (B,Hk,N,d), element strides
  const void* v;
  long long ksb, ksh, ksn, vsb, vsh, vsn;
  const int* lengths;  // (B) rows of each sample
  const int* starts;   // (B) position of row 0, or null: 0
  LowbitCache kc, vc;
  int B, Hk, N, d, window, n_sink;
  int first;  // workgroup of the launch's first (launch_slices.h)
};

struct CacheReadArgs {
  LowbitCache kc, vc;  // plain caches: codes are elements, strides in elements
  const int* lengths;  // (B) positions that have entered
  void* k;             // (B,Hk,S,d) contiguous
  void* v;
  float* mask;  // (B,S)
  int B, Hk, d, window, n_sink;
  int first;
};

struct LowbitDecodeArgs {
  const void* q;  // (B,H,d), element strides
  const void* k;  // (B,Hk,d)
  const void* v;
  long long qsb, qsh, ksb, ksh, vsb, vsh;
  LowbitCache kc, vc;
  const int* lengths;  // (B) position of the token; < 0: none
  const float* table;
  RelSpec rel;
  int B, H, Hk, d, window, n_sink;
  float scale;
  bool q_fast;  // the queries' rows are 16-byte aligned, d a multiple of 8
  void* o;      // (B,H,d) contiguous
  float* part;  // [B*H][n_split][2 + DP]: reference, sum, output of a split (n_split > 1)
  int waves;           // of a workgroup
  int n_split, chunk;  // slots of a split, a multiple of 32
};

// How a decode is cut up: query heads and waves of a workgroup, splits of the cache and slots of one.
struct LowbitPlan {
  int heads, waves, n_split, chunk;
};

struct RowCodesArgs {
  const void* x;  // (M,K), element stride
  long long xs;
  int8_t* codes;  // (M, cs), zeros from K on; 16-byte aligned, cs a multiple of 16
  long long cs;
  float* scale;  // (M)
  long long M;
  int K;
};

// Kernels of the product: codes formed in it, or by a kernel before; tiles of 16 or 32 tokens and 16 rows of weights, or square.
enum Int8Form { I8_OWN_8, I8_OWN_16, I8_OWN_32, I8_FEW_16, I8_FEW_32, I8_TILE_64, I8_TILE_128, I8_TILE_256 };

struct Int8LinearArgs {
  const void* x;    // (M,K) tokens, element stride (I8_OWN_*)
  long long xs;
  const int8_t* a;  // (M, as) codes of the tokens, zeros from K on; as a multiple of 128
  const float* a_scale;
  const int8_t* w;  // (N, ws) codes of the weights
  const float* w_scale;
  const void* bias;  // (N) or null
  void* y;           // (M,N)
  long long as, ws;
  int M, K, N;
  int first;  // 16 rows of weights of the launch's first workgroup (I8_OWN_*, I8_FEW_*)
};

}  // namespace dfl
