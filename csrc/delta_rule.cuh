// Gated delta rule, chunked (training, prefill) and token by token (decoding): delta_rule.cu, delta_step.cu.
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
  bool wide;           // rows of q, k, v and the output's gradient start on 16-byte boundaries
};

struct DeltaGates {
  HeadRows a, b;  // (B, T, H): width 1
  const void *a_log, *dt_bias;
  Elem a_log_type, dt_bias_type;
};

// What the forward leaves for the backward. n = (batch * H + head) * chunks + chunk. 16-bit planes: a value is the sum of
// its two halves, hi and lo, which keeps 16 bits of its significand.
struct DeltaKept {
  __nv_bfloat16* solve;   // (n, 2, 64, 64): the inverse of I + L diag(beta)
  __nv_bfloat16* attend;  // (n, 2, 64, 64): P, lower triangle and diagonal
  __nv_bfloat16* writes;  // (n, 2, 64, dv): V', what each token writes
  __nv_bfloat16* states;  // ((batch * H + head) * (chunks + 1) + chunk, 2, dk, dv): the state before each chunk, and the last
  float2* total;          // (n, 64): sum of log-decays from the chunk's start, in two parts
  float* beta;            // (n, 64)
  float *rk, *rq;         // ((batch * Hk + key head) * chunks + chunk, 64): reciprocal lengths, that of q times scale
};

struct DeltaFwd {
  DeltaDims d;
  HeadRows q, k, v;
  DeltaGates g;
  DeltaKept keep;
  const float* first;  // (B, H, dk, dv) or null
  float* last;         // (B, H, dk, dv) or null
  void* out;           // (B, T, H, dv)
};

struct DeltaBwd {
  DeltaDims d;
  HeadRows q, k, v;
  DeltaGates g;
  DeltaKept keep;
  const void* g_out;      // (B, T, H, dv)
  const float* g_last;    // (B, H, dk, dv) or null
  __nv_bfloat16* dstates;  // (n, 2, dk, dv): the gradient of the state after each chunk
  __nv_bfloat16* dreads;   // (n, 2, 64, dv): the values' gradient before it is rounded
  float* part;             // (n, 2): the chunk's sums for a_log and dt_bias
  void *dq, *dk, *dv, *da, *db, *da_log, *ddt_bias;
  float* dfirst;           // (B, H, dk, dv) or null
};

struct DeltaStep {
  DeltaDims d;
  HeadRows q, k, v;
  DeltaGates g;
  float* state;  // (B, H, dk, dv)
  long long ssb, ssh;
  void* out;  // (B, T, H, dv)
};

int delta_rule_fwd(const DeltaFwd& a, cudaStream_t s);  // the kernels launched
int delta_rule_bwd(const DeltaBwd& a, cudaStream_t s);
void delta_step(const DeltaStep& a, cudaStream_t s);

}  // namespace bw
