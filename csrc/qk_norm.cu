// RMS norm of each query and key head, then the rotation of its first R elements by position.
//
//     r = rsqrt(mean x^2 + eps),  n = x r,  y = n w,
//     (y_i, y_{i+R/2}) -> (y_i cos - y_{i+R/2} sin, y_{i+R/2} cos + y_i sin)     i < R / 2
// Backward, with dy the gradient rotated by the opposite angle:
//     dw = sum over tokens and heads of dy n,    dx = r (w dy - n mean(w dy n)).
// Arithmetic is fp32; the result is rounded once.
#include "qk_norm.cuh"

#include "logit_loss.cuh"

namespace bw {
namespace {

constexpr int kWarps = 8;
constexpr int kPairs = kMaxHeadDim / 64;  // element pairs of one lane

__device__ __forceinline__ float weight_at(const void* w, Elem t, int i) {
  if (t == Elem::kF32) return reinterpret_cast<const float*>(w)[i];
  if (t == Elem::kBF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[i]);
  return __half2float(reinterpret_cast<const __half*>(w)[i]);
}

__device__ __forceinline__ void weight_put(void* w, Elem t, int i, float v) {
  if (t == Elem::kF32)
    reinterpret_cast<float*>(w)[i] = v;
  else if (t == Elem::kBF16)
    reinterpret_cast<__nv_bfloat16*>(w)[i] = __float2bfloat16_rn(v);
  else
    reinterpret_cast<__half*>(w)[i] = __float2half_rn(v);
}

// Pair j of a head: elements (j, j + R/2) are rotated together, the rest go by twos without rotation.
__device__ __forceinline__ void pair_at(int j, int half, int& lo, int& hi) {
  if (j < half) {
    lo = j;
    hi = j + half;
  } else {
    lo = 2 * j;
    hi = 2 * j + 1;
  }
}

// The row of the tables for a token; one outside them is reported and held to them.
__device__ __forceinline__ int table_row(const QkNormArgs& a, int b, int t) {
  const int64_t p = a.positions != nullptr ? a.positions[b * a.pb + t * a.pt] : t;
  if (p >= 0 && p < a.table) return (int)p;
  *a.err = kErrArgument;
  return p < 0 ? 0 : a.table - 1;
}

// One head for each warp.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) qk_norm_fwd_kernel(QkNormArgs a) {
  const int lane = threadIdx.x & 31, heads = a.q.H + a.k.H;
  const long long item = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (item >= (long long)a.B * a.T * heads) return;
  int h = (int)(item % heads);
  const long long token = item / heads;
  const int b = (int)(token / a.T), t = (int)(token % a.T);
  const bool is_q = h < a.q.H;
  if (!is_q) h -= a.q.H;
  const HeadTensor& X = is_q ? a.q : a.k;
  const T* x = reinterpret_cast<const T*>(X.in) + b * X.sb + t * X.st + h * X.sh;
  T* out = reinterpret_cast<T*>(X.out) + (token * X.H + h) * a.D;
  const int half = a.R / 2, pos = table_row(a, b, t);
  float u[kPairs], v[kPairs], ss = 0.f;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const int j = lane + 32 * i;
    u[i] = v[i] = 0.f;
    if (j < a.D / 2) {
      int lo, hi;
      pair_at(j, half, lo, hi);
      u[i] = ElemOf<T>::up(x[lo]);
      v[i] = ElemOf<T>::up(x[hi]);
      ss += u[i] * u[i] + v[i] * v[i];
    }
  }
  const float r = rsqrtf(lanes_sum(ss) / a.D + a.eps);
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const int j = lane + 32 * i;
    if (j < a.D / 2) {
      int lo, hi;
      pair_at(j, half, lo, hi);
      float y0 = u[i] * r * weight_at(X.w, a.wtype, lo), y1 = v[i] * r * weight_at(X.w, a.wtype, hi);
      if (j < half) {
        const float c = a.cos[(long long)pos * half + j], s = a.sin[(long long)pos * half + j];
        const float z0 = y0 * c - y1 * s;
        y1 = y1 * c + y0 * s;
        y0 = z0;
      }
      out[lo] = ElemOf<T>::down(y0);
      out[hi] = ElemOf<T>::down(y1);
    }
  }
}

// CTAs [0, q_blocks) take q's heads, the others k's; each keeps one weight gradient.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) qk_norm_bwd_kernel(QkNormGradArgs g) {
  __shared__ float sum[kMaxHeadDim];
  const QkNormArgs& a = g.f;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = a.R / 2;
  const bool is_q = (int)blockIdx.x < g.q_blocks;
  const HeadTensor& X = is_q ? a.q : a.k;
  const int block = is_q ? blockIdx.x : blockIdx.x - g.q_blocks, blocks = is_q ? g.q_blocks : g.k_blocks;
  const T* grad = reinterpret_cast<const T*>(is_q ? g.gq : g.gk);
  const long long gb = is_q ? g.gqb : g.gkb, gt = is_q ? g.gqt : g.gkt, gh = is_q ? g.gqh : g.gkh;
  const long long items = (long long)a.B * a.T * X.H;
  for (int i = threadIdx.x; i < a.D; i += blockDim.x) sum[i] = 0.f;
  __syncthreads();
  float dw0[kPairs], dw1[kPairs];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) dw0[i] = dw1[i] = 0.f;
  for (long long item = (long long)block * kWarps + warp; item < items; item += (long long)blocks * kWarps) {
    const int h = (int)(item % X.H);
    const long long token = item / X.H;
    const int b = (int)(token / a.T), t = (int)(token % a.T);
    const T* x = reinterpret_cast<const T*>(X.in) + b * X.sb + t * X.st + h * X.sh;
    const T* gr = grad == nullptr ? nullptr : grad + b * gb + t * gt + h * gh;
    T* out = reinterpret_cast<T*>(X.out) + item * a.D;
    const int pos = table_row(a, b, t);
    float u[kPairs], v[kPairs], d0[kPairs], d1[kPairs], ss = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const int j = lane + 32 * i;
      u[i] = v[i] = d0[i] = d1[i] = 0.f;
      if (j < a.D / 2) {
        int lo, hi;
        pair_at(j, half, lo, hi);
        u[i] = ElemOf<T>::up(x[lo]);
        v[i] = ElemOf<T>::up(x[hi]);
        ss += u[i] * u[i] + v[i] * v[i];
        float e0 = gr == nullptr ? 0.f : ElemOf<T>::up(gr[lo]), e1 = gr == nullptr ? 0.f : ElemOf<T>::up(gr[hi]);
        if (j < half) {
          const float c = a.cos[(long long)pos * half + j], s = a.sin[(long long)pos * half + j];
          const float z0 = e0 * c + e1 * s;
          e1 = e1 * c - e0 * s;
          e0 = z0;
        }
        d0[i] = e0;
        d1[i] = e1;
        dot += e0 * weight_at(X.w, a.wtype, lo) * u[i] + e1 * weight_at(X.w, a.wtype, hi) * v[i];
      }
    }
    const float r = rsqrtf(lanes_sum(ss) / a.D + a.eps);
    const float mean = lanes_sum(dot) * r / a.D;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const int j = lane + 32 * i;
      if (j < a.D / 2) {
        int lo, hi;
        pair_at(j, half, lo, hi);
        const float n0 = u[i] * r, n1 = v[i] * r;
        dw0[i] += d0[i] * n0;
        dw1[i] += d1[i] * n1;
        out[lo] = ElemOf<T>::down(r * (d0[i] * weight_at(X.w, a.wtype, lo) - n0 * mean));
        out[hi] = ElemOf<T>::down(r * (d1[i] * weight_at(X.w, a.wtype, hi) - n1 * mean));
      }
    }
  }
  for (int w = 0; w < kWarps; ++w) {  // in order, so that sums repeat
    if (warp == w) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const int j = lane + 32 * i;
        if (j < a.D / 2) {
          int lo, hi;
          pair_at(j, half, lo, hi);
          sum[lo] += dw0[i];
          sum[hi] += dw1[i];
        }
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < a.D; i += blockDim.x) g.part[(long long)blockIdx.x * a.D + i] = sum[i];
}

// CTA (i, 0 or 1): element 32 i + lane of one weight's gradient; warps share the CTAs' sums, added in order.
__global__ void __launch_bounds__(256) qk_weight_sum_kernel(QkNormGradArgs g) {
  __shared__ float red[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
  const int first = blockIdx.y == 0 ? 0 : g.q_blocks, n = blockIdx.y == 0 ? g.q_blocks : g.k_blocks;
  float v = 0.f;
  if (e < g.f.D)
    for (int k = warp; k < n; k += 8) v += g.part[(long long)(first + k) * g.f.D + e];
  red[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && e < g.f.D) {
    v = 0.f;
    for (int k = 0; k < 8; ++k) v += red[k][lane];
    weight_put(blockIdx.y == 0 ? g.dqw : g.dkw, g.f.wtype, e, v);
  }
}

}  // namespace

void qk_norm_blocks(const QkNormArgs& a, int* q_blocks, int* k_blocks) {
  const long long tokens = (long long)a.B * a.T, most = 148 * 8;
  const long long q = (tokens * a.q.H + kWarps - 1) / kWarps, k = (tokens * a.k.H + kWarps - 1) / kWarps;
  const long long qs = most * a.q.H / (a.q.H + a.k.H), ks = most - qs;
  *q_blocks = (int)(q < qs ? (q < 1 ? 1 : q) : (qs < 1 ? 1 : qs));
  *k_blocks = (int)(k < ks ? (k < 1 ? 1 : k) : (ks < 1 ? 1 : ks));
}

void qk_norm_fwd(const QkNormArgs& a, cudaStream_t s) {
  const long long items = (long long)a.B * a.T * (a.q.H + a.k.H);
  if (items == 0) return;
  const unsigned grid = (unsigned)((items + kWarps - 1) / kWarps);
  if (a.type == Elem::kBF16)
    qk_norm_fwd_kernel<__nv_bfloat16><<<grid, kWarps * 32, 0, s>>>(a);
  else if (a.type == Elem::kF16)
    qk_norm_fwd_kernel<__half><<<grid, kWarps * 32, 0, s>>>(a);
  else
    qk_norm_fwd_kernel<float><<<grid, kWarps * 32, 0, s>>>(a);
}

void qk_norm_bwd(const QkNormGradArgs& g, cudaStream_t s) {
  const unsigned grid = (unsigned)(g.q_blocks + g.k_blocks);
  if (g.f.type == Elem::kBF16)
    qk_norm_bwd_kernel<__nv_bfloat16><<<grid, kWarps * 32, 0, s>>>(g);
  else if (g.f.type == Elem::kF16)
    qk_norm_bwd_kernel<__half><<<grid, kWarps * 32, 0, s>>>(g);
  else
    qk_norm_bwd_kernel<float><<<grid, kWarps * 32, 0, s>>>(g);
  qk_weight_sum_kernel<<<dim3((g.f.D + 31) / 32, 2), 256, 0, s>>>(g);
}

}  // namespace bw
