// Element types of the post-training kernels: 16-byte vectors of bf16, fp16 or fp32 with
// fp32 arithmetic in between, and the warp reductions they share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace bw {

enum class Elem : int { kBF16 = 0, kF16 = 1, kF32 = 2 };

#ifdef __CUDACC__

template <typename T>
struct ElemOf;

template <>
struct ElemOf<__nv_bfloat16> {
  static constexpr uint32_t kNegInf = 0xff80u;
  static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
};

template <>
struct ElemOf<__half> {
  static constexpr uint32_t kNegInf = 0xfc00u;
  static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
};

template <>
struct ElemOf<float> {
  static constexpr uint32_t kNegInf = 0xff800000u;
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
};

// Elements of a 16-byte vector.
template <typename T>
constexpr int kVecOf = 16 / (int)sizeof(T);

// Two elements of a 32-bit word (one for fp32), converted together: single conversions run at a fraction of the rate.
__device__ __forceinline__ void word_up(uint32_t w, float* f, __nv_bfloat16) {
  f[0] = __uint_as_float(w << 16);
  f[1] = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void word_up(uint32_t w, float* f, __half) {
  const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w));
  f[0] = p.x;
  f[1] = p.y;
}
__device__ __forceinline__ void word_up(uint32_t w, float* f, float) { f[0] = __uint_as_float(w); }

__device__ __forceinline__ uint32_t word_down(const float* f, __nv_bfloat16) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(f[0], f[1]);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t word_down(const float* f, __half) {
  const __half2 p = __floats2half2_rn(f[0], f[1]);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t word_down(const float* f, float) { return __float_as_uint(f[0]); }

// An access of 4, 8 or 16 bytes as words, and its elements in fp32.
__device__ __forceinline__ void words_of(const uint4& r, uint32_t* w) {
  w[0] = r.x;
  w[1] = r.y;
  w[2] = r.z;
  w[3] = r.w;
}
__device__ __forceinline__ void words_of(const uint2& r, uint32_t* w) {
  w[0] = r.x;
  w[1] = r.y;
}
__device__ __forceinline__ void words_of(const uint32_t& r, uint32_t* w) { w[0] = r; }
__device__ __forceinline__ void of_words(uint4& r, const uint32_t* w) { r = make_uint4(w[0], w[1], w[2], w[3]); }
__device__ __forceinline__ void of_words(uint2& r, const uint32_t* w) { r = make_uint2(w[0], w[1]); }
__device__ __forceinline__ void of_words(uint32_t& r, const uint32_t* w) { r = w[0]; }

template <typename T, typename Raw>
__device__ __forceinline__ void raw_up(const Raw& r, float* f) {
  constexpr int kWords = sizeof(Raw) / 4, kPer = 4 / sizeof(T);
  uint32_t w[kWords];
  words_of(r, w);
#pragma unroll
  for (int i = 0; i < kWords; ++i) word_up(w[i], f + i * kPer, T());
}

template <typename T, typename Raw>
__device__ __forceinline__ Raw raw_down(const float* f) {
  constexpr int kWords = sizeof(Raw) / 4, kPer = 4 / sizeof(T);
  uint32_t w[kWords];
#pragma unroll
  for (int i = 0; i < kWords; ++i) w[i] = word_down(f + i * kPer, T());
  Raw r;
  of_words(r, w);
  return r;
}

template <typename V>
__device__ __forceinline__ V lanes_sum(V v, int width = 32) {
  for (int o = width / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

#endif  // __CUDACC__

}  // namespace bw
