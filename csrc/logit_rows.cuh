// Rows of logits as the kernels of the losses and of the token scores read them: 16-byte vectors whatever a row starts
// at, maxima and sums of exponentials over a warp or a CTA.
#pragma once

#include <cmath>
#include <cstring>

#include "logit_loss.cuh"
#include "tc_common.cuh"

namespace bw {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row as 16-byte vectors on 16-byte boundaries: vector j holds elements [j N - shift, j N - shift + N).
// Vectors that reach over an end of the row are read and written an element at a time.
template <typename T>
struct RowSpan {
  static constexpr int N = kVecOf<T>;
  const T* row;
  int shift, nv, V;

  __device__ RowSpan(const T* p, int v) : row(p), V(v) {
    shift = (int)((reinterpret_cast<uintptr_t>(p) % 16) / sizeof(T));
    nv = (V + shift + N - 1) / N;
  }
  __device__ __forceinline__ int first(int j) const { return j * N - shift; }
  // Whether vectors [j0, j0 + n) all belong to the row whole.
  __device__ __forceinline__ bool inner(int j0, int n) const {
    return (j0 > 0 || shift == 0) && j0 + n <= (V + shift) / N;
  }
  __device__ __forceinline__ bool whole(int lo) const { return lo >= 0 && lo + N <= V; }
  __device__ __forceinline__ const uint4* vec(int j) const { return reinterpret_cast<const uint4*>(row - shift) + j; }
  // Vector j; elements outside the row are -inf. kLast: nothing reads it again soon.
  template <bool kLast>
  __device__ __forceinline__ uint4 load(int j) const {
    const int lo = first(j);
    if (lo >= 0 && lo + N <= V) {
      const uint4* p = reinterpret_cast<const uint4*>(row + lo);
      return kLast ? __ldcs(p) : __ldcg(p);
    }
    constexpr uint32_t kFill = sizeof(T) == 2 ? ElemOf<T>::kNegInf * 0x10001u : ElemOf<T>::kNegInf;
    uint32_t w[4] = {kFill, kFill, kFill, kFill};
    if (j < nv) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (lo + i >= 0 && lo + i < V) put(w, i, row[lo + i]);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ void put(uint32_t* w, int i, T v) {
    if constexpr (sizeof(T) == 2) {
      uint16_t b;
      memcpy(&b, &v, 2);
      w[i / 2] = (w[i / 2] & (i & 1 ? 0xffffu : 0xffff0000u)) | (uint32_t)b << (i & 1 ? 16 : 0);
    } else {
      memcpy(&w[i], &v, 4);
    }
  }
};

template <typename T>
__device__ __forceinline__ void store_vec(T* row, int V, int lo, const uint4& v, bool aligned) {
  constexpr int N = kVecOf<T>;
  if (aligned && lo >= 0 && lo + N <= V) {
    __stcs(reinterpret_cast<uint4*>(row + lo), v);
    return;
  }
  float f[N];
  raw_up<T>(v, f);  // exact: the values came from T
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (lo + i >= 0 && lo + i < V) row[lo + i] = ElemOf<T>::down(f[i]);
}

// What the terms of a part with maximum m are taken off: 0 where all of it is -inf, so that its terms are 0.
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// The label's log-probability. Its own logit goes without the factor log2(e), which would take the type's lowest value,
// what a mask may have put there, to -inf.
__device__ __forceinline__ float label_logp_of(float xy, float base, float inv_temp, float log2_s) {
  return (xy - base) * inv_temp - kLn2 * log2_s;
}
__device__ __forceinline__ float label_logp(float xy, float base, float inv_temp, float s) {
  return label_logp_of(xy, base, inv_temp, log2f(s));
}

// The larger of each element of two words; a NaN is passed over here and found again in the sum.
__device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b, __nv_bfloat16) {
  const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b, __half) {
  const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b, float) {
  return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
}

template <typename T, int K>
__device__ __forceinline__ float max_of(const uint4 (&r)[K]) {
  uint32_t m = word_max(word_max(r[0].x, r[0].y, T()), word_max(r[0].z, r[0].w, T()), T());
#pragma unroll
  for (int k = 1; k < K; ++k)
    m = word_max(m, word_max(word_max(r[k].x, r[k].y, T()), word_max(r[k].z, r[k].w, T()), T()), T());
  float f[4 / sizeof(T)];
  word_up(m, f, T());
  return sizeof(T) == 2 ? fmaxf(f[0], f[4 / sizeof(T) - 1]) : f[0];
}

// 2^((x - base) c) of a vector's elements, by twos.
template <typename T>
__device__ __forceinline__ void powers(const uint4& r, float base, float c, float2 (&e)[kVecOf<T> / 2]) {
  constexpr int N = kVecOf<T>;
  float f[N];
  raw_up<T>(r, f);
  const float2 off = make_float2(-base, -base), cc = make_float2(c, c);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float2 t = __fmul2_rn(__fadd2_rn(make_float2(f[2 * i], f[2 * i + 1]), off), cc);
    e[i] = make_float2(ex2(t.x), ex2(t.y));
  }
}

template <typename T, int K>
__device__ __forceinline__ float sum_of(const uint4 (&r)[K], float base, float c) {
  float2 s = make_float2(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float2 e[kVecOf<T> / 2];
    powers<T>(r[k], base, c, e);
#pragma unroll
    for (int i = 0; i < kVecOf<T> / 2; ++i) s = __fadd2_rn(s, e[i]);
  }
  return s.x + s.y;
}

// coef (onehot(y) - softmax) of a vector whose first element is `lo`: k = -coef / s.
template <typename T>
__device__ __forceinline__ uint4 grad_of(const uint4& r, int lo, int y, float base, float c, float k, float coef) {
  constexpr int N = kVecOf<T>;
  float2 e[N / 2];
  powers<T>(r, base, c, e);
  float f[N];
  const float2 kk = make_float2(k, k);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float2 g = __fmul2_rn(e[i], kk);
    f[2 * i] = g.x;
    f[2 * i + 1] = g.y;
  }
  if ((unsigned)(y - lo) < (unsigned)N) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lo + i == y) f[i] += coef;
  }
  return raw_down<T, uint4>(f);
}

// The maximum and the sum of a warp's parts (m, s), s counting 2^((x - m) c); in every lane.
__device__ __forceinline__ void merge_warp(float& m, float& s, float c) {
  float M = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  // A part that saw only -inf has s = 0 (or NaN from a NaN logit): its factor only has to be finite.
  s = lanes_sum(s * (m == -INFINITY ? 1.f : ex2((m - M) * c)));
  m = M;
}

// The same over the threads of a row.
template <int kGroup>
__device__ __forceinline__ void merge_group(float& m, float& s, float c, float2* parts) {
  constexpr int kW = kGroup / 32;
  merge_warp(m, s, c);
  if constexpr (kW > 1) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) parts[threadIdx.x >> 5] = make_float2(m, s);
    __syncthreads();
    const float2 p = lane < kW ? parts[lane] : make_float2(-INFINITY, 0.f);
    m = p.x;
    s = p.y;
    merge_warp(m, s, c);
  }
}

constexpr int kUnroll = 4;  // vectors of a thread in one step

// The row's label, or -1 where the row does not count.
__device__ __forceinline__ int row_label(const LogitRows& r, long long row) {
  const int64_t y = r.labels[row];
  if (y == r.ignore) return -1;
  if (y < 0 || y >= r.V) {
    if ((threadIdx.x & 31) == 0) report_error(r.err, kErrBadArg);
    return -1;
  }
  return (int)y;
}

template <typename T>
__device__ __forceinline__ const T* row_ptr(const LogitRows& r, long long row) {
  const long long b = row / r.T, t = row - b * r.T;
  return reinterpret_cast<const T*>(r.x) + b * r.sb + t * r.st;
}

// ---------------------------------------------------------------- row statistics
// Rows go to groups of kGroup threads: whole CTAs, or the warps of a CTA of four (a short row leaves a wider group
// waiting on its own barriers, and an SM takes 32 CTAs at most).
template <int kGroup>
struct Place {
  static constexpr int kRows = kGroup == 32 ? 4 : 1, kThreads = kGroup * kRows;
  static __device__ __forceinline__ int tid() { return kRows > 1 ? threadIdx.x & 31 : threadIdx.x; }
  static __device__ __forceinline__ long long row() {
    return kRows > 1 ? (long long)blockIdx.x * kRows + (threadIdx.x >> 5) : blockIdx.x;
  }
};

// kUnroll vectors of a thread from vector j on, kStride apart; `whole`: all of the row. kLast: nothing reads them again soon.
template <typename T, int kStride, bool kLast>
__device__ __forceinline__ void fetch(const RowSpan<T>& span, int j, bool whole, uint4 (&to)[kUnroll]) {
  if (whole) {
    const uint4* p = span.vec(j);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) to[u] = kLast ? __ldcs(p + u * kStride) : __ldcg(p + u * kStride);
  } else {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) to[u] = span.template load<kLast>(j + u * kStride);
  }
}

// Takes vectors into a thread's running maximum and sum.
template <typename T>
__device__ __forceinline__ void take(const uint4 (&v)[kUnroll], float c, float& m, float& s) {
  const float top = max_of<T>(v);
  if (top > m) {
    s *= m == -INFINITY ? 1.f : ex2((m - top) * c);
    m = top;
  }
  s += sum_of<T>(v, base_of(m), c);
}

// The maximum and the sum of a row, in every thread of its group: one pass with a running maximum and sum in each.
template <typename T, int kGroup>
__device__ __forceinline__ void row_stats(const RowSpan<T>& span, float c, float& m, float& s, float2* parts) {
  constexpr int kHold = kGroup * kUnroll;
  m = -INFINITY;
  s = 0.f;
  const int tid = Place<kGroup>::tid();
  for (int j = tid; j < span.nv; j += kHold) {
    uint4 v[kUnroll];
    fetch<T, kGroup, false>(span, j, span.inner(j - tid, kHold), v);
    take<T>(v, c, m, s);
  }
  merge_group<kGroup>(m, s, c, parts);
}

template <typename T, int kGroup>
__device__ __forceinline__ void zero_row(T* out, int V) {
  const RowSpan<T> span(out, V);
  for (int j = Place<kGroup>::tid(); j < span.nv; j += kGroup) store_vec<T>(out, V, span.first(j), make_uint4(0, 0, 0, 0), true);
}

}  // namespace
}  // namespace bw
