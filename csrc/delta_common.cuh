// What the kernels of the gated delta rule share: gates, matrix tiles in two 16-bit halves, loads of head rows.
#pragma once

#include <cuda_fp16.h>

#include "delta_rule.cuh"

namespace bw {
namespace {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ float load_any(const void* p, Elem type, long long i) {
  if (type == Elem::kBF16) return __bfloat162float(reinterpret_cast<const bf16*>(p)[i]);
  if (type == Elem::kF16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return reinterpret_cast<const float*>(p)[i];
}

__device__ __forceinline__ void store_any(void* p, Elem type, long long i, float v) {
  if (type == Elem::kBF16) reinterpret_cast<bf16*>(p)[i] = __float2bfloat16_rn(v);
  else if (type == Elem::kF16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else reinterpret_cast<float*>(p)[i] = v;
}

__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

struct Gate {
  float log_decay, rate, slope;  // g = -rate softplus(x), slope = sigmoid(x)
};

// A log-decay below -1e4 closes the gate like any other below -104, and keeps sums of 64 of them exact to 1e-10.
__device__ __forceinline__ Gate gate_of(float a, float a_log, float dt_bias) {
  const float x = a + dt_bias;
  const float soft = x > 20.f ? x : log1pf(expf(x));
  const float rate = expf(a_log);
  const float g = -rate * soft;
  return Gate{g < -1e4f ? -1e4f : g, rate, sigmoid(x)};
}

}  // namespace
}  // namespace bw
