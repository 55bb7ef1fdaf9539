// Argument blocks of the sequence operators (window attention, its rolling cache, the
// relative position bias), shared by the kernels and the C-ABI layer.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "window_geometry.h"

namespace dfl {

struct WinArgs {
  const void* q;  // (B,H,M,d), element strides qsb/qsh/qsn, unit inner stride
  const void* k;  // (B,Hk,N,d), element strides ksb/ksh/ksn
  const void* v;  // (B,Hk,N,d), element strides vsb/vsh/vsn
  long long qsb, qsh, qsn;
  long long ksb, ksh, ksn;
  long long vsb, vsh, vsn;
  const float* mask;   // (B,N) or null; 0 = masked
  const float* table;  // (H, rel.buckets()) or null
  RelSpec rel;
  int B, H, Hk, M, N, d;
  int window, n_sink, causal;
  float scale;
  void* o;     // (B,H,M,d) contiguous
  void* o_rest;  // (B,H,M,d) or null; bf16: sum p~ v / sum p~ - o with the rounded weights p~, where !win_few_keys
  float* lse;  // (B,H,M) base-2 log of the row sums; LSE_EMPTY on rows that see nothing
  // backward
  const void* go;  // (B,H,M,d) contiguous
  void* dq;        // (B,H,M,d) contiguous
  void* dk;        // (B,Hk,N,d) contiguous
  void* dv;
  float* dtable;    // (H, buckets) or null
  float* rowd;      // [B*H][M][2]: D_i and the row's factor (0 where the row has one key, else 1)
  float* sink_part; // [B*Hk][n_chunks + 1][n_sink][2][DP] partial dK / dV of the first tokens (n_chunks > 0)
  float* kv_part;   // [kv_split][B*Hk][N][2][DP] partial dK / dV (kv_split > 1)
  float* tab_part;  // [B*H*q blocks][buckets]
  int kv_split;     // parts of a key tile's queries, each in a workgroup of its own
  int n_chunks;     // query chunks of the first tokens' gradients; 0: nothing lies outside the band
  int chunk;        // queries of a chunk
};
constexpr float LSE_EMPTY = 1.0e30f;

// Rolling cache of n_sink + window slots a (b, key head): position p < n_sink lies in slot p, any other in slot
// n_sink + (p - n_sink) % window.
struct CacheFillArgs {
  const void* k;  // (B,Hk,N,d) new rows, element strides
  const void* v;
  long long ksb, ksh, ksn, vsb, vsh, vsn;
  const int* lengths;  // (B) rows of each sample
  void* kc;            // (B,Hk,n_sink + window,d), element strides
  void* vc;
  long long kcsb, kcsh, kcsn, vcsb, vcsh, vcsn;
  int B, Hk, N, d, window, n_sink;
};

struct DecodeArgs {
  const void* q;  // (B,H,d), element strides
  const void* k;  // (B,Hk,d) the token's own key and value, element strides
  const void* v;
  long long qsb, qsh, ksb, ksh, vsb, vsh;
  void* kc;  // as in CacheFillArgs
  void* vc;
  long long kcsb, kcsh, kcsn, vcsb, vcsh, vcsn;
  const int* lengths;  // (B) position of the token; < 0: no token, zero output, cache untouched
  const float* table;
  RelSpec rel;
  int B, H, Hk, d, window, n_sink;
  float scale;
  void* o;      // (B,H,d) contiguous
  float* part;  // [B*H][n_split][2 + DP]: reference, sum, output of a split (n_split > 1)
  int n_split, chunk;  // slots of a split
};

struct RelBiasArgs {
  const float* table;  // (H, buckets)
  RelSpec rel;
  const int* q_pos;  // (B,M) or null: position i + N - M
  const int* k_pos;  // (B,N) or null: position j
  int B, H, M, N;
  void* out;            // (B,H,M,N)
  const void* grad;     // (B,H,M,N)
  float* dtable;        // (H, buckets)
  float* part;          // [B*H][n_part][buckets]
  int n_part;
};

}  // namespace dfl
