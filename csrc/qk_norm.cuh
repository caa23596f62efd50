// RMS norm of every query and key head with the position rotation in the same pass (qk_norm.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "elem.cuh"

namespace bw {

constexpr int kMaxHeadDim = 512;

struct HeadTensor {
  const void* in;
  long long sb, st, sh;  // element strides of batch, token and head; the head's elements are contiguous
  void* out;             // (B, T, H, D) contiguous
  const void* w;         // (D)
  int H;
};

struct QkNormArgs {
  HeadTensor q, k;
  Elem type, wtype;
  const float *cos, *sin;    // (table, R / 2)
  const int64_t* positions;  // (B, T) with strides, or null: the token's index
  long long pb, pt;
  int B, T, D, R, table;     // R: rotated elements at the head's start
  float eps;
  int* err;
};

// Backward: q.in / k.in are the inputs of the forward, q.out / k.out their gradients.
struct QkNormGradArgs {
  QkNormArgs f;
  const void *gq, *gk;  // gradients of the outputs; null: zero
  long long gqb, gqt, gqh, gkb, gkt, gkh;
  float* part;          // (blocks, D): weight gradient sums of each CTA
  int q_blocks, k_blocks;
  void *dqw, *dkw;      // (D) in the weights' type
};

void qk_norm_fwd(const QkNormArgs& a, cudaStream_t s);
void qk_norm_bwd(const QkNormGradArgs& a, cudaStream_t s);
// CTAs that the backward wants for q and for k.
void qk_norm_blocks(const QkNormGradArgs& g, int* q_blocks, int* k_blocks);

}  // namespace bw
