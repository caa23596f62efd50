// Balance loss of an expert router, forward and backward.
//
// With p = softmax(x) of the N tokens that count, f_e the choices of expert e per token and
// P_e the mean of p_e:
//     loss = E sum_e f_e P_e + z mean(lse^2)
//     dx_ne = g [ E p_ne (f_e - sum_j f_j p_nj) + 2 z lse_n p_ne ] / N        (f is a constant)
#include "router_balance.cuh"

#include <cmath>

#include "tc_common.cuh"

namespace bw {
namespace {

constexpr int kWarps = 8;

// Order-preserving key: larger values first, a NaN before all, -0 equal to 0. 0 is left for "taken".
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  if (v != v) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One token for each warp at a time; lane l holds experts l, l + 32, ...
template <typename T, int kPer>
__global__ void __launch_bounds__(kWarps * 32) balance_fwd_kernel(BalanceArgs a) {
  extern __shared__ float smem[];
  float* sum_p = smem;
  int* hist = reinterpret_cast<int*>(smem + a.E + 1);
  const int g = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e <= a.E; e += blockDim.x) {
    sum_p[e] = 0.f;
    hist[e] = 0;
  }
  __syncthreads();
  float acc[kPer], z = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
  int tokens = 0;
  for (int n = blockIdx.x * kWarps + warp; n < a.N; n += gridDim.x * kWarps) {
    const long long at = (long long)g * a.N + n;
    if (a.mask != nullptr && !a.mask[at]) continue;
    ++tokens;
    const T* x = reinterpret_cast<const T*>(a.x) + g * a.sg + n * a.sn;
    float v[kPer], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = lane + 32 * i;
      v[i] = e < a.E ? ElemOf<T>::up(x[e]) : -INFINITY;
      top = fmaxf(top, v[i]);
    }
    if (a.ids == nullptr) {
      uint32_t key[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) key[i] = lane + 32 * i < a.E ? order_key(v[i]) : 0u;
      for (int k = 0; k < a.K; ++k) {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) best = max(best, key[i]);
        best = __reduce_max_sync(0xffffffffu, best);
        int e = INT32_MAX;
#pragma unroll
        for (int i = kPer - 1; i >= 0; --i)
          if (key[i] == best) e = lane + 32 * i;
        e = __reduce_min_sync(0xffffffffu, e);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (e == lane + 32 * i) key[i] = 0;
        if (lane == 0) atomicAdd(hist + e, 1);
      }
    } else {
      for (int k = lane; k < a.K; k += 32) {
        const int64_t e = a.ids[at * a.K + k];
        if (e >= 0 && e < a.E)
          atomicAdd(hist + e, 1);
        else
          report_error(a.err, kErrBadArg);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      v[i] = lane + 32 * i < a.E ? __expf(v[i] - top) : 0.f;
      s += v[i];
    }
    s = lanes_sum(s);
    const float inv = 1.f / s, lse = top + __logf(s);
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] += v[i] * inv;
    z += lse * lse;
  }
  for (int w = 0; w < kWarps; ++w) {  // in order, so that sums repeat
    if (warp == w) {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (lane + 32 * i < a.E) sum_p[lane + 32 * i] += acc[i];
      if (lane == 0) {
        sum_p[a.E] += z;
        hist[a.E] += tokens;
      }
    }
    __syncthreads();
  }
  const long long base = ((long long)g * a.chunks + blockIdx.x) * (a.E + 1);
  for (int e = threadIdx.x; e <= a.E; e += blockDim.x) {
    a.part[base + e] = sum_p[e];
    a.part_count[base + e] = hist[e];
  }
}

// One CTA for each group: adds the chunks in order.
__global__ void __launch_bounds__(256) balance_finish_kernel(BalanceArgs a) {
  __shared__ double red[8];
  const int g = blockIdx.x;
  const long long base = (long long)g * a.chunks * (a.E + 1);
  long long tokens = 0;
  double zz = 0;
  for (int k = 0; k < a.chunks; ++k) {
    tokens += a.part_count[base + (long long)k * (a.E + 1) + a.E];
    zz += a.part[base + (long long)k * (a.E + 1) + a.E];
  }
  const double inv = 1.0 / (tokens > 0 ? (double)tokens : 1.0);
  double dot = 0;
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
    long long c = 0;
    double p = 0;
    for (int k = 0; k < a.chunks; ++k) {
      c += a.part_count[base + (long long)k * (a.E + 1) + e];
      p += a.part[base + (long long)k * (a.E + 1) + e];
    }
    a.counts[(long long)g * a.E + e] = c;
    a.share[(long long)g * (a.E + 1) + e] = (float)(c * inv);
    dot += c * inv * p;
  }
  dot = lanes_sum(dot);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = dot;
  __syncthreads();
  if (threadIdx.x == 0) {
    dot = 0;
    for (int k = 0; k < 8; ++k) dot += red[k];
    a.loss[g] = (float)(a.E * dot * inv + (a.z_coef != 0.f ? a.z_coef * zz * inv : 0.0));
    a.share[(long long)g * (a.E + 1) + a.E] = (float)inv;
  }
}

template <typename T, int kPer>
__global__ void __launch_bounds__(kWarps * 32) balance_bwd_kernel(BalanceGradArgs b) {
  const BalanceArgs& a = b.f;
  const int g = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float* share = a.share + (long long)g * (a.E + 1);
  const float scale = b.g_loss[g * b.g_stride] * share[a.E];
  float f[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) f[i] = lane + 32 * i < a.E ? share[lane + 32 * i] * a.E : 0.f;
  for (int n = blockIdx.x * kWarps + warp; n < a.N; n += gridDim.x * kWarps) {
    const long long at = (long long)g * a.N + n;
    T* out = reinterpret_cast<T*>(b.out) + at * a.E;
    if (a.mask != nullptr && !a.mask[at]) {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (lane + 32 * i < a.E) out[lane + 32 * i] = ElemOf<T>::down(0.f);
      continue;
    }
    const T* x = reinterpret_cast<const T*>(a.x) + g * a.sg + n * a.sn;
    float v[kPer], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      v[i] = lane + 32 * i < a.E ? ElemOf<T>::up(x[lane + 32 * i]) : -INFINITY;
      top = fmaxf(top, v[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float s = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      v[i] = lane + 32 * i < a.E ? __expf(v[i] - top) : 0.f;
      s += v[i];
      dot += v[i] * f[i];
    }
    s = lanes_sum(s);
    dot = lanes_sum(dot);
    const float inv = 1.f / s, lse = top + __logf(s), shift = 2.f * a.z_coef * lse - dot * inv;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lane + 32 * i < a.E) out[lane + 32 * i] = ElemOf<T>::down(scale * (v[i] * inv) * (f[i] + shift));
  }
}

template <typename T, int kPer>
void launch_fwd(const BalanceArgs& a, cudaStream_t s) {
  const size_t smem = 2 * (a.E + 1) * sizeof(float);
  balance_fwd_kernel<T, kPer><<<dim3(a.chunks, a.G), kWarps * 32, smem, s>>>(a);
}

template <typename T, int kPer>
void launch_bwd(const BalanceGradArgs& b, cudaStream_t s) {
  balance_bwd_kernel<T, kPer><<<dim3(b.f.chunks, b.f.G), kWarps * 32, 0, s>>>(b);
}

template <typename T>
void fwd_of(const BalanceArgs& a, cudaStream_t s) {
  if (a.E <= 64) return launch_fwd<T, 2>(a, s);
  if (a.E <= 256) return launch_fwd<T, 8>(a, s);
  launch_fwd<T, 32>(a, s);
}

template <typename T>
void bwd_of(const BalanceGradArgs& b, cudaStream_t s) {
  if (b.f.E <= 64) return launch_bwd<T, 2>(b, s);
  if (b.f.E <= 256) return launch_bwd<T, 8>(b, s);
  launch_bwd<T, 32>(b, s);
}

}  // namespace

void balance_fwd(const BalanceArgs& a, cudaStream_t s) {
  if (a.type == Elem::kBF16)
    fwd_of<__nv_bfloat16>(a, s);
  else if (a.type == Elem::kF16)
    fwd_of<__half>(a, s);
  else
    fwd_of<float>(a, s);
  balance_finish_kernel<<<a.G, 256, 0, s>>>(a);
}

void balance_bwd(const BalanceGradArgs& b, cudaStream_t s) {
  if (b.f.type == Elem::kBF16)
    bwd_of<__nv_bfloat16>(b, s);
  else if (b.f.type == Elem::kF16)
    bwd_of<__half>(b, s);
  else
    bwd_of<float>(b, s);
}

}  // namespace bw
