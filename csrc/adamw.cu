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
// Sums of squares are fp32: a gradient whose square passes its range (1e20 or so) leaves an infinite root. The codes of its block of
// 256 then have an infinite scale, and the next step makes NaN of them, as an infinite gradient does at once.
//
// What bounds it: a bf16 weight moves 22 bytes with moments in 32 bits, at the rate of a copy: 486 M weights take 1,590 us. With
// moments in 8 bits it moves 10, in 1,180 us: 60 instructions an element fill 70 % of the issue slots while memory runs at 60 % of a
// copy's rate; 64 registers leave 32 warps to an SM, too few to fill either.
#include "adamw.cuh"

#include <cuda_fp8.h>

#include <cstring>

namespace bw {
namespace {

constexpr int kThreads = 256, kN = 8;  // elements of a thread's step
constexpr float kF8Max = 448.f, kF8Tiny = 0.001953125f;

// Square root and reciprocal to an ulp or two, in a few instructions where the compiler's correctly rounded ones take ten. The root
// takes numbers below the normal range, squares of gradients under 1e-19; the reciprocal is of a root, 3e-23 at least, or of eps.
__device__ __forceinline__ float root_of(float v) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float inverse_of(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// The weight after a step with the new m and the root of the new v.
__device__ __forceinline__ float stepped(const AdamwStep& a, float p, float m, float root) {
  return fmaf(-a.size, m * inverse_of(fmaf(root, a.inv_root2, a.eps)), a.keep * p);
}

__device__ __forceinline__ void update(const AdamwStep& a, float& p, float g, float& m, float& v) {
  m = fmaf(a.beta1, m, a.one_beta1 * g);
  v = fmaf(a.beta2, v, a.one_beta2 * g * g);
  p = stepped(a, p, m, root_of(v));
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

// The tensor that chunk blockIdx.x belongs to: the lanes of each warp look at the first chunks side by side.
template <int N>
__device__ __forceinline__ int tensor_of(const AdamwTable<N>& a) {
  const int lane = threadIdx.x & 31;
  int at = -1;
  for (int i = 0; i < a.s.count; i += 32) {
    const bool past = i + lane >= a.s.count || a.first[i + lane] > blockIdx.x;
    const unsigned after = __ballot_sync(0xffffffffu, past);
    if (after == 0) {
      at = i + 31;
      continue;
    }
    if (after != 0xffffffffu) at = i + __ffs(after) - 2;
    break;
  }
  return at;
}

template <typename P, typename G, int N>
__global__ void __launch_bounds__(kThreads) adamw32_kernel(const __grid_constant__ AdamwTable<N> a) {
  const int at = tensor_of(a);
  const AdamwTensor& t = a.t[at];
  const long long from = (long long)(blockIdx.x - a.first[at]) * a.s.chunk, size = t.n < 0 ? -t.n : t.n;
  const int n = (int)min((long long)a.s.chunk, size - from);
  P* p = reinterpret_cast<P*>(t.p) + from;
  const G* g = reinterpret_cast<const G*>(t.g) + from;
  float *m = reinterpret_cast<float*>(t.m) + from, *v = reinterpret_cast<float*>(t.v) + from;
  int done = 0;
  if (t.n > 0) {
    done = n / kN * kN;
#pragma unroll 2
    for (int i = threadIdx.x * kN; i < done; i += kThreads * kN) {
      float pf[kN], gf[kN], mf[kN], vf[kN];
      load8(p + i, pf);
      load8(g + i, gf);
      load8(m + i, mf);
      load8(v + i, vf);
#pragma unroll
      for (int k = 0; k < kN; ++k) update(a.s, pf[k], gf[k], mf[k], vf[k]);
      store8(p + i, pf);
      store8(m + i, mf);
      store8(v + i, vf);
    }
  }
#pragma unroll 4
  for (int i = done + threadIdx.x; i < n; i += kThreads) {
    float pf = ElemOf<P>::up(p[i]), mf = m[i], vf = v[i];
    update(a.s, pf, ElemOf<G>::up(g[i]), mf, vf);
    p[i] = ElemOf<P>::down(pf);
    m[i] = mf;
    v[i] = vf;
  }
}

// An e4m3 code's exponent and significand as the low exponent bits and the significand of an fp32 number are that number
// times 2^-120, small codes included. 2^120 is a product of its own, which is exact: with it in the scale, scales from 256 on would
// be infinite. The codes of NaN never come: a NaN goes into the scale.
constexpr float kF8Up = 1329227995784915872903807060280344576.f;  // 2^120

// Code k of a word, with and without a sign.
__device__ __forceinline__ float f8_up(uint32_t w, int k) {
  return __uint_as_float((uint32_t)((int)(w << (24 - 8 * k)) >> 4) & 0x87f00000u);
}
__device__ __forceinline__ float f8_up_plus(uint32_t w, int k) {
  return __uint_as_float((k < 3 ? w << (20 - 8 * (k < 3 ? k : 0)) : w >> 4) & 0x07f00000u);
}

__device__ __forceinline__ uint32_t f8_down(float x, float y) {
  return __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float max_nan(float x, float y) {
  float z;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
  return z;
}

// The scale of a block whose largest magnitude is `top`, and its reciprocal. Magnitudes near the end of fp32's range keep a
// scale whose reciprocal is finite.
__device__ __forceinline__ float scale_of(float top, float& inv) {
  const float s = top == 0.f ? 0.f : max_nan(top * (1.f / kF8Max), 1e-37f);
  inv = top == 0.f ? 0.f : __frcp_rn(s);
  return s;
}

__device__ __forceinline__ float2 two(float x) { return make_float2(x, x); }

// Sums of products that are rounded first: no product joins the addition as a fused one.
__device__ __forceinline__ float2 sum_of(float2 x, float2 y) { return make_float2(__fadd_rn(x.x, y.x), __fadd_rn(x.y, y.y)); }

// Square roots of two values, to half an ulp or so (an ulp or two below the normal range, where the rest is rounded to its steps):
// the estimate of the reciprocal root and a step of Newton's method on the largest number at most; what an infinity has over
// that comes on top. 0 stays 0.
__device__ __forceinline__ float2 roots_of(float2 v) {
  float2 r, w;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(w.x) : "f"(v.x), "f"(3.4028234663852886e38f));
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(w.y) : "f"(v.y), "f"(3.4028234663852886e38f));
  asm("rsqrt.approx.f32 %0, %1;" : "=f"(r.x) : "f"(fmaxf(w.x, 1.4e-45f)));
  asm("rsqrt.approx.f32 %0, %1;" : "=f"(r.y) : "f"(fmaxf(w.y, 1.4e-45f)));
  const float2 s = __fmul2_rn(w, r), over = __fadd2_rn(v, make_float2(-w.x, -w.y));
  const float2 rest = __ffma2_rn(make_float2(-s.x, -s.y), s, w);
  return __fadd2_rn(__ffma2_rn(rest, __fmul2_rn(r, two(0.5f)), s), over);
}

// Two quotients x / scale to half an ulp: the product with the reciprocal and what remains of x. Codes next to a border
// then fall as those of a division do.
__device__ __forceinline__ float2 ratios_of(float2 x, float scale, float inv) {
  const float2 q = __fmul2_rn(x, two(inv));
  return __ffma2_rn(__ffma2_rn(make_float2(-q.x, -q.y), two(scale), x), two(inv), q);
}

// A root that is not zero is at least the smallest code.
__device__ __forceinline__ float root_code(float ratio, float r) { return fmaxf(ratio, r > 0.f ? kF8Tiny : 0.f); }

// What a lane holds of a block: eight elements side by side where whole vectors may be moved, else 32 apart.
template <typename P, typename G>
struct Block {
  uint4 p[sizeof(P) / 2], g[sizeof(G) / 2];
  uint2 m, v;
  float sm, sv;
};

template <typename T>
__device__ __forceinline__ void fetch8(uint4 (&to)[sizeof(T) / 2], const T* x, bool wide, int n) {
  const int lane = threadIdx.x & 31;
  if (wide) {
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k) to[k] = __ldcs(reinterpret_cast<const uint4*>(x + lane * kN) + k);
    return;
  }
  T e[kN];
#pragma unroll
  for (int k = 0; k < kN; ++k) {
    const int i = k * 32 + lane;
    e[k] = i < n ? x[i] : ElemOf<T>::down(0.f);
  }
  memcpy(to, e, sizeof(e));
}

__device__ __forceinline__ uint2 fetch_codes(const uint8_t* x, bool wide, int n) {
  const int lane = threadIdx.x & 31;
  if (wide) return __ldcs(reinterpret_cast<const uint2*>(x) + lane);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < kN; ++k) {
    const int i = k * 32 + lane;
    if (i < n) w[k / 4] |= (uint32_t)x[i] << (k % 4 * 8);
  }
  return make_uint2(w[0], w[1]);
}

// What becomes codes is computed as the formulas stand, each operation rounded by itself: a value next to a border between two
// codes falls as it does for anyone else, and states stay comparable over many steps, in which one code may decide a scale.
//
// A warp takes blocks of 256 elements, whose scales are its own maxima; the next block is on its way while one is computed.
template <typename P, typename G, int N>
__global__ void __launch_bounds__(kThreads, 4) adamw8_kernel(const __grid_constant__ AdamwTable<N> a) {
  const int at = tensor_of(a);
  const AdamwTensor& t = a.t[at];
  const long long size = t.n < 0 ? -t.n : t.n, blocks = (size + kMomentBlock - 1) / kMomentBlock;
  const int per = a.s.chunk / kMomentBlock, lane = threadIdx.x & 31;
  const bool aligned = t.n > 0;
  P* const p = reinterpret_cast<P*>(t.p);
  const G* const g = reinterpret_cast<const G*>(t.g);
  uint8_t *const m = reinterpret_cast<uint8_t*>(t.m), *const v = reinterpret_cast<uint8_t*>(t.v);
  float* const scale = t.scale;
  const long long first = (long long)(blockIdx.x - a.first[at]) * per, end = min(blocks, first + per);
  const auto fetch = [&](long long block, Block<P, G>& b) {
    const long long from = block * kMomentBlock;
    const int n = (int)min((long long)kMomentBlock, size - from);
    const bool wide = aligned && n == kMomentBlock;
    fetch8<P>(b.p, p + from, wide, n);
    fetch8<G>(b.g, g + from, wide, n);
    b.m = fetch_codes(m + from, wide, n);
    b.v = fetch_codes(v + from, wide, n);
    b.sm = scale[block];
    b.sv = scale[blocks + block];
  };
  long long block = first + (threadIdx.x >> 5);
  if (block >= end) return;
  Block<P, G> now, next;
  fetch(block, now);
#pragma unroll 1
  for (; block < end; block += kThreads / 32) {
    if (block + kThreads / 32 < end) fetch(block + kThreads / 32, next);
    float pf[kN], gf[kN], mf[kN], vf[kN];
#pragma unroll
    for (int k = 0; k < (int)sizeof(P) / 2; ++k) raw_up<P>(now.p[k], pf + k * 4);
#pragma unroll
    for (int k = 0; k < (int)sizeof(G) / 2; ++k) raw_up<G>(now.g[k], gf + k * 4);
    const uint32_t mw[2] = {now.m.x, now.m.y}, vw[2] = {now.v.x, now.v.y};
    float top_m = 0.f, top_r = 0.f;
#pragma unroll
    for (int k = 0; k < kN; k += 2) {
      const float2 g2 = make_float2(gf[k], gf[k + 1]);
      const float2 v_code = make_float2(f8_up_plus(vw[k / 4], k % 4), f8_up_plus(vw[k / 4], k % 4 + 1));
      const float2 m_code = make_float2(f8_up(mw[k / 4], k % 4), f8_up(mw[k / 4], k % 4 + 1));
      const float2 r = __fmul2_rn(__fmul2_rn(v_code, two(kF8Up)), two(now.sv));
      const float2 old = __fmul2_rn(__fmul2_rn(m_code, two(kF8Up)), two(now.sm));
      const float2 m2 = sum_of(__fmul2_rn(two(a.s.beta1), old), __fmul2_rn(two(a.s.one_beta1), g2));
      const float2 v2 = sum_of(__fmul2_rn(two(a.s.beta2), __fmul2_rn(r, r)), __fmul2_rn(__fmul2_rn(two(a.s.one_beta2), g2), g2));
      const float2 root = roots_of(v2), den = __ffma2_rn(root, two(a.s.inv_root2), two(a.s.eps));
      const float2 q = __fmul2_rn(m2, make_float2(inverse_of(den.x), inverse_of(den.y)));
      const float2 p2 = __ffma2_rn(two(-a.s.size), q, __fmul2_rn(two(a.s.keep), make_float2(pf[k], pf[k + 1])));
      pf[k] = p2.x;
      pf[k + 1] = p2.y;
      mf[k] = m2.x;
      mf[k + 1] = m2.y;
      vf[k] = root.x;
      vf[k + 1] = root.y;
      top_m = max_nan(max_nan(top_m, fabsf(m2.x)), fabsf(m2.y));
      top_r = max_nan(max_nan(top_r, root.x), root.y);
    }
    const long long from = block * kMomentBlock;
    const int n = (int)min((long long)kMomentBlock, size - from);
    const bool wide = aligned && n == kMomentBlock;
    if (wide) {
      store8(p + from + lane * kN, pf);
    } else {
#pragma unroll
      for (int k = 0; k < kN; ++k)
        if (k * 32 + lane < n) p[from + k * 32 + lane] = ElemOf<P>::down(pf[k]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      top_m = max_nan(top_m, __shfl_xor_sync(0xffffffffu, top_m, o));
      top_r = max_nan(top_r, __shfl_xor_sync(0xffffffffu, top_r, o));
    }
    float im, ir;
    const float new_m = scale_of(top_m, im), new_r = scale_of(top_r, ir);
    if (lane == 0) {
      scale[block] = new_m;
      scale[blocks + block] = new_r;
    }
    uint32_t mc[2] = {0, 0}, vc[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < kN; k += 2) {
      const float2 x = ratios_of(make_float2(mf[k], mf[k + 1]), new_m, im), y = ratios_of(make_float2(vf[k], vf[k + 1]), new_r, ir);
      mc[k / 4] |= f8_down(x.x, x.y) << (k % 4 * 8);
      vc[k / 4] |= f8_down(root_code(y.x, vf[k]), root_code(y.y, vf[k + 1])) << (k % 4 * 8);
    }
    if (wide) {
      __stcs(reinterpret_cast<uint2*>(m + from) + lane, make_uint2(mc[0], mc[1]));
      __stcs(reinterpret_cast<uint2*>(v + from) + lane, make_uint2(vc[0], vc[1]));
    } else {
#pragma unroll
      for (int k = 0; k < kN; ++k) {
        const int i = k * 32 + lane;
        if (i >= n) continue;
        m[from + i] = (uint8_t)(mc[k / 4] >> (k % 4 * 8));
        v[from + i] = (uint8_t)(vc[k / 4] >> (k % 4 * 8));
      }
    }
    now = next;
  }
}

template <typename P, typename G, int N>
void launch(const AdamwTable<N>& a, bool bits8, cudaStream_t s) {
  if (bits8) adamw8_kernel<P, G, N><<<a.s.chunks, kThreads, 0, s>>>(a);
  else adamw32_kernel<P, G, N><<<a.s.chunks, kThreads, 0, s>>>(a);
}

template <int N>
void launch(const AdamwTable<N>& a, Elem p, Elem g, bool bits8, cudaStream_t s) {
  if (p == Elem::kF32) return launch<float, float>(a, bits8, s);
  if (p == Elem::kBF16) {
    if (g == Elem::kF32) return launch<__nv_bfloat16, float>(a, bits8, s);
    return launch<__nv_bfloat16, __nv_bfloat16>(a, bits8, s);
  }
  if (g == Elem::kF32) return launch<__half, float>(a, bits8, s);
  launch<__half, __half>(a, bits8, s);
}

}  // namespace

void adamw_step(const AdamwTable<kAdamwMany>& a, Elem p, Elem g, bool bits8, cudaStream_t s) {
  if (a.s.count > kAdamwFew) return launch(a, p, g, bits8, s);
  AdamwTable<kAdamwFew> few;
  few.s = a.s;
  std::memcpy(few.first, a.first, sizeof(few.first));
  std::memcpy(few.t, a.t, sizeof(few.t));
  launch(few, p, g, bits8, s);
}

}  // namespace bw
