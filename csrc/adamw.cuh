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
  long long n;   // negative: -n elements that cannot be moved as whole vectors
};

// The table travels as a kernel's argument (32,764 bytes at most), so a step copies nothing to the device beforehand.
// A step of few tensors takes the small one: 15.5 us instead of 17.5 for 20 tensors.
constexpr int kAdamwFew = 32, kAdamwMany = 512;

struct AdamwStep {
  int count;
  int chunk;  // elements of a CTA, a multiple of 2048
  unsigned chunks;
  // one_beta1 = 1 - b1, negative where the step maximizes
  // p <- keep p - size m / (sqrt(v) inv_root2 + eps)
  float beta1, beta2, one_beta1, one_beta2, keep, size, inv_root2, eps;
};

template <int N>
struct AdamwTable {
  AdamwStep s;
  unsigned first[N];  // the first chunk of each tensor
  AdamwTensor t[N];
};

// Elements of a CTA for a step of `total`: the more there are, the more a CTA takes before the next one has to find its tensor
// and fill its pipeline again; a few CTAs for each SM at least. 125,000 weights take 2.8 us in chunks of 2048 and 7.5 in chunks
// of 32768.
inline int adamw_chunk(int64_t total, bool bits8) {
  const int most = bits8 ? 32768 : 8192;
  int chunk = 2048;
  while (chunk < most && total / (4 * chunk) >= 148 * 8) chunk *= 4;
  return chunk;
}

void adamw_step(const AdamwTable<kAdamwMany>& a, Elem p_type, Elem g_type, bool bits8, cudaStream_t s);

}  // namespace bw
