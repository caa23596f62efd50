// AdamW step of many tensors in one launch, moments in 32 or 8 bits (adamw.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "elem.cuh"

namespace bw {

constexpr int kMomentBlock = 256;  // elements that share a scale of an 8-bit moment

struct AdamwTensor {
  void* p;
  const void* g;
  void *m, *v;   // fp32, or e4m3 codes
  float* scale;  // (2, blocks): scales of m and of the root of v; null for fp32 moments
  long long n;
  unsigned first;    // the first chunk of this tensor
  unsigned aligned;  // whole vectors may be moved
};

// The table travels as a kernel's argument (32,764 bytes at most), so a step copies nothing to the device beforehand.
constexpr int kAdamwTensors = 480;
constexpr int kAdamwChunk = 8192;  // elements of a CTA

struct AdamwTable {
  AdamwTensor t[kAdamwTensors];
  int count;
  unsigned chunks;
  // p <- keep p - size m / (sqrt(v) inv_root2 + eps)
  float beta1, beta2, one_beta1, one_beta2, keep, size, inv_root2, eps, sign;
};

void adamw_step(const AdamwTable& a, Elem p_type, Elem g_type, bool bits8, cudaStream_t s);

}  // namespace bw
