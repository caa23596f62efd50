// AdamW step of many tensors:
//     m <- b1 m + (1 - b1) g,   v <- b2 v + (1 - b2) g^2,
//     p <- (1 - lr wd) p - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps),
// all in fp32 and each result rounded once.
//
// Moments in 8 bits: 256 elements share a scale, the largest magnitude among them over 448, and each is an e4m3 code of
// its ratio to the scale. What stands for v is its root: a step divides by it, its relative error is then the code's
// (2^-4) whatever the gradients' size, and 17 octaves of codes span 34 of v. A root that is not zero takes the smallest
// code at least, so that no weight is divided by eps alone because its neighbours' gradients are large. The step
// itself uses the moments before they are rounded to codes.
//
// What bounds it: memory. A bf16 weight moves 22 bytes with moments in 32 bits and 10 with moments in 8.
#include "adamw.cuh"

#include <cuda_fp8.h>

namespace bw {
namespace {

constexpr int kThreads = 256, kN = 8;  // elements of a thread's step
constexpr float kF8Max = 448.f, kF8Tiny = 0.001953125f;

struct Moments {
  float m[kN], v[kN];
};

__device__ __forceinline__ void update(const AdamwTable& a, float& p, float g, float& m, float& v) {
  g *= a.sign;
  m = fmaf(a.beta1, m, a.one_beta1 * g);
  v = fmaf(a.beta2, v, a.one_beta2 * g * g);
  const float root = sqrtf(v);
  p = fmaf(-a.size, __fdividef(m, fmaf(root, a.inv_root2, a.eps)), a.keep * p);
}

// n consecutive elements as fp32, by 16-byte accesses.
template <typename T>
__device__ __forceinline__ void load8(const T* x, float (&f)[kN]) {
  const uint4* p = reinterpret_cast<const uint4*>(x);
  if constexpr (sizeof(T) == 2) {
    raw_up<T>(__ldcs(p), f);
  } else {
    raw_up<T>(__ldcs(p), f);
    raw_up<T>(__ldcs(p + 1), f + 4);
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* x, const float (&f)[kN]) {
  uint4* p = reinterpret_cast<uint4*>(x);
  if constexpr (sizeof(T) == 2) {
    __stcs(p, raw_down<T, uint4>(f));
  } else {
    __stcs(p, raw_down<T, uint4>(f));
    __stcs(p + 1, raw_down<T, uint4>(f + 4));
  }
}

__device__ __forceinline__ const AdamwTensor& tensor_of(const AdamwTable& a, unsigned chunk) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.t[mid].first <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return a.t[lo];
}

template <typename P, typename G>
__global__ void __launch_bounds__(kThreads) adamw32_kernel(const __grid_constant__ AdamwTable a) {
  const AdamwTensor& t = tensor_of(a, blockIdx.x);
  const long long from = (long long)(blockIdx.x - t.first) * kAdamwChunk;
  const int n = (int)min((long long)kAdamwChunk, t.n - from);
  P* p = reinterpret_cast<P*>(t.p) + from;
  const G* g = reinterpret_cast<const G*>(t.g) + from;
  float *m = reinterpret_cast<float*>(t.m) + from, *v = reinterpret_cast<float*>(t.v) + from;
  int done = 0;
  if (t.aligned) {
    done = n / kN * kN;
#pragma unroll 2
    for (int i = threadIdx.x * kN; i < done; i += kThreads * kN) {
      float pf[kN], gf[kN], mf[kN], vf[kN];
      load8(p + i, pf);
      load8(g + i, gf);
      load8(m + i, mf);
      load8(v + i, vf);
#pragma unroll
      for (int k = 0; k < kN; ++k) update(a, pf[k], gf[k], mf[k], vf[k]);
      store8(p + i, pf);
      store8(m + i, mf);
      store8(v + i, vf);
    }
  }
#pragma unroll 4
  for (int i = done + threadIdx.x; i < n; i += kThreads) {
    float pf = ElemOf<P>::up(p[i]), mf = m[i], vf = v[i];
    update(a, pf, ElemOf<G>::up(g[i]), mf, vf);
    p[i] = ElemOf<P>::down(pf);
    m[i] = mf;
    v[i] = vf;
  }
}

__device__ __forceinline__ float2 f8_up(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

__device__ __forceinline__ uint32_t f8_down(float x, float y) {
  return __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
}

// The scale of a block whose largest magnitude is `top`, and what its values are multiplied by. Magnitudes near the
// end of fp32's range keep a scale whose reciprocal is finite.
__device__ __forceinline__ float scale_of(float top, float& inv) {
  const float s = top > 0.f ? fmaxf(top * (1.f / kF8Max), 1e-37f) : 0.f;
  inv = top > 0.f ? __frcp_rn(s) : 0.f;
  return s;
}

__device__ __forceinline__ float root_code(float r, float inv) { return r > 0.f ? fmaxf(r * inv, kF8Tiny) : r * inv; }

// A warp takes a block of 256 elements: the scales are its own maxima.
template <typename P, typename G>
__global__ void __launch_bounds__(kThreads) adamw8_kernel(const __grid_constant__ AdamwTable a) {
  const AdamwTensor& t = tensor_of(a, blockIdx.x);
  const unsigned chunk = blockIdx.x - t.first;
  const long long blocks = (t.n + kMomentBlock - 1) / kMomentBlock;
  constexpr int kPer = kAdamwChunk / kMomentBlock;
  const int lane = threadIdx.x & 31;
  const bool aligned = t.aligned != 0;
#pragma unroll 1
  for (int w = threadIdx.x >> 5; w < kPer; w += kThreads / 32) {
    const long long block = (long long)chunk * kPer + w;
    if (block >= blocks) return;
    const long long from = block * kMomentBlock;
    const bool whole = from + kMomentBlock <= t.n;
    P* p = reinterpret_cast<P*>(t.p) + from;
    const G* g = reinterpret_cast<const G*>(t.g) + from;
    uint8_t *m = reinterpret_cast<uint8_t*>(t.m) + from, *v = reinterpret_cast<uint8_t*>(t.v) + from;
    const float sm = t.scale[block], sv = t.scale[blocks + block];
    const bool wide = whole && aligned;
    const int n = (int)min((long long)kMomentBlock, t.n - from);
    float pf[kN], gf[kN], mf[kN], vf[kN];
    if (wide) {
      load8(p + lane * kN, pf);
      load8(g + lane * kN, gf);
      const uint2 mc = __ldcs(reinterpret_cast<const uint2*>(m) + lane), vc = __ldcs(reinterpret_cast<const uint2*>(v) + lane);
      const uint32_t mw[2] = {mc.x, mc.y}, vw[2] = {vc.x, vc.y};
#pragma unroll
      for (int k = 0; k < kN; k += 2) {
        const float2 x = f8_up(mw[k / 4] >> (k % 4 * 8) & 0xffffu), y = f8_up(vw[k / 4] >> (k % 4 * 8) & 0xffffu);
        mf[k] = x.x;
        mf[k + 1] = x.y;
        vf[k] = y.x;
        vf[k + 1] = y.y;
      }
    } else {  // a lane's elements are 32 apart
#pragma unroll
      for (int k = 0; k < kN; ++k) {
        const int i = k * 32 + lane;
        const bool in = i < n;
        pf[k] = in ? ElemOf<P>::up(p[i]) : 0.f;
        gf[k] = in ? ElemOf<G>::up(g[i]) : 0.f;
        mf[k] = in ? f8_up(m[i]).x : 0.f;
        vf[k] = in ? f8_up(v[i]).x : 0.f;
      }
    }
    float top_m = 0.f, top_r = 0.f;
#pragma unroll
    for (int k = 0; k < kN; ++k) {
      const float r = vf[k] * sv;
      mf[k] *= sm;
      vf[k] = r * r;
      update(a, pf[k], gf[k], mf[k], vf[k]);
      vf[k] = sqrtf(vf[k]);
      top_m = fmaxf(top_m, fabsf(mf[k]));
      top_r = fmaxf(top_r, vf[k]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      top_m = fmaxf(top_m, __shfl_xor_sync(0xffffffffu, top_m, o));
      top_r = fmaxf(top_r, __shfl_xor_sync(0xffffffffu, top_r, o));
    }
    float im, ir;
    const float new_m = scale_of(top_m, im), new_r = scale_of(top_r, ir);
    if (lane == 0) {
      t.scale[block] = new_m;
      t.scale[blocks + block] = new_r;
    }
    if (wide) {
      uint32_t mw[2] = {0, 0}, vw[2] = {0, 0};
#pragma unroll
      for (int k = 0; k < kN; k += 2) {
        mw[k / 4] |= f8_down(mf[k] * im, mf[k + 1] * im) << (k % 4 * 8);
        vw[k / 4] |= f8_down(root_code(vf[k], ir), root_code(vf[k + 1], ir)) << (k % 4 * 8);
      }
      store8(p + lane * kN, pf);
      __stcs(reinterpret_cast<uint2*>(m) + lane, make_uint2(mw[0], mw[1]));
      __stcs(reinterpret_cast<uint2*>(v) + lane, make_uint2(vw[0], vw[1]));
    } else {
#pragma unroll
      for (int k = 0; k < kN; ++k) {
        const int i = k * 32 + lane;
        if (i >= n) continue;
        p[i] = ElemOf<P>::down(pf[k]);
        m[i] = (uint8_t)f8_down(mf[k] * im, 0.f);
        v[i] = (uint8_t)f8_down(root_code(vf[k], ir), 0.f);
      }
    }
  }
}

template <typename P, typename G>
void launch(const AdamwTable& a, bool bits8, cudaStream_t s) {
  if (bits8) adamw8_kernel<P, G><<<a.chunks, kThreads, 0, s>>>(a);
  else adamw32_kernel<P, G><<<a.chunks, kThreads, 0, s>>>(a);
}

}  // namespace

void adamw_step(const AdamwTable& a, Elem p, Elem g, bool bits8, cudaStream_t s) {
  if (p == Elem::kF32) return launch<float, float>(a, bits8, s);
  if (p == Elem::kBF16) {
    if (g == Elem::kF32) return launch<__nv_bfloat16, float>(a, bits8, s);
    return launch<__nv_bfloat16, __nv_bfloat16>(a, bits8, s);
  }
  if (g == Elem::kF32) return launch<__half, float>(a, bits8, s);
  launch<__half, __half>(a, bits8, s);
}

}  // namespace bw
