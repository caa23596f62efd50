// Gated delta rule, chunked (training, prefill) and token by token (decoding): delta_prepare.cu, delta_state.cu and delta_inputs.cu; delta_step.cu.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "elem.cuh"

namespace bw {

constexpr int kChunk = 64;         // tokens of a chunk
constexpr int kMostKeyDim = 128;   // elements of a key head
constexpr int kMostGroup = 8;      // value heads of a key head: a cluster in the backward

// (B, T, heads, width) with a contiguous last axis and any other strides (in elements).
struct HeadRows {
  const void* p;
  long long sb, st, sh;
};

struct DeltaDims {
  int B, T, Hk, H, dk, dv, chunks;
  Elem type;           // of q, k, v, a, b and the output
  float scale;         // of the queries
  bool wide;           // rows of q and k start on 16-byte boundaries
  // Value elements are cut into slices, lanes of tensor memory: of 64 where a head has no more, or where two parts of
  // q and k beside a state of 128 leave no room for 128.
  int slice, slices;
};

struct DeltaGates {
  HeadRows a, b;  // (B, T, H): width 1
  const void *a_log, *dt_bias;
  Elem a_log_type, dt_bias_type;
};

// What the forward leaves for the backward, as tiles (delta_tiles.cuh) of two halves unless said otherwise.
// n = (batch * H + head) * chunks + chunk, m = (batch * Hk + key head) * chunks + chunk; kp is dk up to 64 or 128.
struct DeltaKept {
  unsigned char *keys, *queries;  // (m): [tokens][kp], one part for each of the type's
  unsigned char* solve;           // (n): [64][64], the inverse of I + L diag(beta)
  unsigned char* attend;          // (n): [64][64], P
  unsigned char* writes;          // (n, slice): [slice][tokens], V'^T; null without a backward
  unsigned char* states;          // (n, slice): [slice][kp], S^T before each chunk; null likewise
  float2* total;                  // (n, 64): sum of log-decays from the chunk's start, in two parts
  float* beta;                    // (n, 64)
  float *rk, *rq;                 // (m, 64): reciprocal lengths, that of q times scale
};

struct DeltaFwd {
  DeltaDims d;
  HeadRows q, k, v;
  DeltaGates g;
  DeltaKept keep;
  const float* first;  // (B, H, dk, dv) or null
  float* last;         // (B, H, dk, dv) or null
  void* out;           // (B, T, H, dv)
  int* err;
};

struct DeltaBwd {
  DeltaDims d;
  HeadRows q, k, v;
  DeltaGates g;
  DeltaKept keep;
  const void* g_out;       // (B, T, H, dv)
  const float* g_last;     // (B, H, dk, dv) or null
  unsigned char* dstates;  // (n, slice): [slice][kp], dS'^T, the gradient of the state after each chunk
  unsigned char* dreads;   // (n, slice): [slice][tokens], dV^T before it is rounded
  unsigned char* douts;    // (n, slice): [slice][tokens], dO^T, one part for each of the type's
  float* part;             // (n, 2): the chunk's sums for a_log and dt_bias
  void *dq, *dk, *dv, *da, *db, *da_log, *ddt_bias;
  float* dfirst;           // (B, H, dk, dv) or null
  int* err;
};

struct DeltaStep {
  DeltaDims d;
  HeadRows q, k, v;
  DeltaGates g;
  float* state;  // (B, H, dk, dv)
  long long ssb, ssh;
  void* out;  // (B, T, H, dv)
  int* err;
};

void delta_prepare(const DeltaFwd& a, cudaStream_t s);
void delta_state(const DeltaFwd& a, cudaStream_t s);
void delta_dstate(const DeltaBwd& a, cudaStream_t s);
void delta_inputs(const DeltaBwd& a, cudaStream_t s);
void delta_step(const DeltaStep& a, cudaStream_t s);

// The kernels launched.
inline int delta_rule_fwd(const DeltaFwd& a, cudaStream_t s) {
  if (a.d.B * a.d.H == 0) return 0;
  if (a.d.chunks > 0) delta_prepare(a, s);
  delta_state(a, s);
  return a.d.chunks > 0 ? 2 : 1;
}
inline int delta_rule_bwd(const DeltaBwd& a, cudaStream_t s) {
  if (a.d.B > 0) delta_dstate(a, s);
  delta_inputs(a, s);
  return (a.d.B > 0) + (a.d.B * a.d.chunks > 0) + 1;
}

}  // namespace bw
