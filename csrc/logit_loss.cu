// Preference and policy losses from logits.
//
// Both need log p(y | row) = x_y - lse(x) of the labelled token of every row that counts, and
// both send back coef (onehot(y) - softmax(x)). In base two with c = log2(e) / temperature and
// m = max(x):
//     s = sum_v 2^((x_v - m) c),   log p = ln 2 ((x_y - m) c - log2 s),   p_v = 2^((x_v - m) c) / s.
// The maximum is taken off before the scaling: x_v c - m c in one step would overflow where a
// mask put the type's lowest value. Sums are fp32 within a row (each thread its share) and fp64
// over a sequence's tokens and over pairs.
//
// A row whose label is ignored is not read: whatever stands there, its log-probability is 0
// and its gradient is 0.
#include "logit_loss.cuh"

#include <cmath>

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
  // Vector j; elements outside the row are -inf.
  __device__ __forceinline__ uint4 load(int j) const {
    const int lo = j * N - shift;
    if (lo >= 0 && lo + N <= V) return __ldg(reinterpret_cast<const uint4*>(row + lo));
    constexpr uint32_t kFill = sizeof(T) == 2 ? ElemOf<T>::kNegInf * 0x10001u : ElemOf<T>::kNegInf;
    uint4 r = make_uint4(kFill, kFill, kFill, kFill);
    T* e = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lo + i >= 0 && lo + i < V) e[i] = row[lo + i];
    return r;
  }
};

template <typename T>
__device__ __forceinline__ void store_vec(T* row, int V, int lo, const uint4& v, bool aligned) {
  constexpr int N = kVecOf<T>;
  if (aligned && lo >= 0 && lo + N <= V) {
    __stcs(reinterpret_cast<uint4*>(row + lo), v);
    return;
  }
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (lo + i >= 0 && lo + i < V) row[lo + i] = e[i];
}

// What the terms of a part with maximum m are taken off: 0 where all of it is -inf, so that its terms are 0.
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

template <int kThreads>
__device__ __forceinline__ void block_max_sum(float& m, float& s, float c, float* red) {
  float M = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kW = kThreads / 32;
  if (lane == 0) red[warp] = M;
  __syncthreads();
  M = red[0];
#pragma unroll
  for (int k = 1; k < kW; ++k) M = fmaxf(M, red[k]);
  // A thread that saw only -inf has s = 0 (or NaN from a NaN logit): its factor only has to be finite.
  s *= m == -INFINITY ? 1.f : ex2((m - M) * c);
  s = lanes_sum(s);
  if (lane == 0) red[32 + warp] = s;
  __syncthreads();
  s = red[32];
#pragma unroll
  for (int k = 1; k < kW; ++k) s += red[32 + k];
  m = M;
}

// The row's label, or -1 where the row does not count.
__device__ __forceinline__ int row_label(const LogitRows& r, long long row) {
  const int64_t y = r.labels[row];
  if (y == r.ignore) return -1;
  if (y < 0 || y >= r.V) {
    if (threadIdx.x == 0) *r.err = kErrArgument;
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
// One CTA for each row, one pass with a running maximum and sum in every thread.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) row_stats_kernel(LogitRows r, float* __restrict__ logps,
                                                             RowStat* __restrict__ stats,
                                                             unsigned* __restrict__ ticket) {
  constexpr int N = kVecOf<T>;
  __shared__ float red[64];
  const long long row = blockIdx.x;
  if (row == 0 && threadIdx.x == 0) *ticket = 0;
  const int y = row_label(r, row);
  if (y < 0) {
    if (threadIdx.x == 0) {
      logps[row] = 0.f;
      stats[row] = RowStat{0.f, 0.f};
    }
    return;
  }
  const T* x = row_ptr<T>(r, row);
  const RowSpan<T> span(x, r.V);
  const float c = kLog2e * r.inv_temp;
  float m = -INFINITY, base = 0.f, s = 0.f;
  for (int j = threadIdx.x; j < span.nv; j += kThreads) {
    float f[N];
    raw_up<T>(span.load(j), f);
    float top = f[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, f[i]);
    if (top > m) {
      s *= m == -INFINITY ? 1.f : ex2((m - top) * c);
      m = base = top;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) s += ex2((f[i] - base) * c);
  }
  block_max_sum<kThreads>(m, s, c, red);
  if (threadIdx.x == 0) {
    base = base_of(m);
    logps[row] = kLn2 * ((ElemOf<T>::up(x[y]) - base) * c - log2f(s));
    stats[row] = RowStat{base, 1.f / s};
  }
}

// ---------------------------------------------------------------- gradient
// One CTA for each row: coef (onehot - softmax) / temperature. A zero coefficient (an ignored row, a clipped token)
// writes zeros without reading the row.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) logit_grad_kernel(LogitGradArgs a) {
  constexpr int N = kVecOf<T>;
  const LogitRows& r = a.rows;
  const long long row = blockIdx.x;
  const long long b = row / r.T, t = row - b * r.T;
  const int y = row_label(r, row);
  T* out = reinterpret_cast<T*>(a.out) + b * a.osb + t * a.ost;
  float coef = 0.f;
  if (y >= 0) {
    const long long i = a.per_row ? row : b;
    if (a.g_loss != nullptr) coef = a.g_loss[a.g_loss_mod ? b % a.g_loss_mod : 0] * a.d[i];
    if (a.g_logps != nullptr) coef += a.g_logps[i];
    if (a.scale != nullptr) coef *= a.scale[b];
    coef *= r.inv_temp;
  }
  if (coef == 0.f) {
    const RowSpan<T> span(out, r.V);
    for (int j = threadIdx.x; j < span.nv; j += kThreads)
      store_vec<T>(out, r.V, j * N - span.shift, make_uint4(0, 0, 0, 0), true);
    return;
  }
  const T* x = row_ptr<T>(r, row);
  const RowSpan<T> span(x, r.V);
  const bool aligned = (int)((reinterpret_cast<uintptr_t>(out) % 16) / sizeof(T)) == span.shift;
  const RowStat st = a.stats[row];
  const float c = kLog2e * r.inv_temp, k = -coef * st.inv_s;
  for (int j = threadIdx.x; j < span.nv; j += kThreads) {
    float f[N];
    raw_up<T>(span.load(j), f);
    const int lo = j * N - span.shift;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      f[i] = ex2((f[i] - st.m) * c) * k;
      if (lo + i == y) f[i] += coef;
    }
    store_vec<T>(out, r.V, lo, raw_down<T, uint4>(f), aligned);
  }
}

// ---------------------------------------------------------------- sums over tokens
__device__ __forceinline__ double block_sum(double v, double* red) {
  v = lanes_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0;
  for (int k = 0; k < (int)blockDim.x / 32; ++k) t += red[k];
  return t;
}

// True in every thread of the CTA that arrives last; what the others wrote before is then visible to it.
__device__ __forceinline__ bool last_block(unsigned* ticket) {
  __shared__ bool last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  __syncthreads();
  __threadfence();
  return last;
}

__device__ __forceinline__ double softplus(double z) { return fmax(z, 0.0) + log1p(exp(-fabs(z))); }

// One CTA for each pair: both sequences' sums, the pair's loss and its derivative; the last CTA adds the losses in order.
__global__ void __launch_bounds__(256) preference_finish_kernel(PreferenceArgs a) {
  __shared__ double red[8];
  const int P = gridDim.x, i = blockIdx.x, T = a.rows.T;
  double total[2], tokens[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const long long base = (long long)(i + h * P) * T;
    double v = 0, n = 0;
    for (int t = threadIdx.x; t < T; t += blockDim.x) {
      v += a.logp_tok[base + t];
      if (a.average) {
        const int64_t y = a.rows.labels[base + t];
        n += y != a.rows.ignore && y >= 0 && y < a.rows.V;
      }
    }
    total[h] = block_sum(v, red);
    tokens[h] = a.average ? fmax(block_sum(n, red), 1.0) : 1.0;
    total[h] /= tokens[h];
  }
  if (threadIdx.x == 0) {
    const double m = (total[0] - a.ref[i]) - (total[1] - a.ref[i + P]);
    const double beta = a.beta, eps = a.smoothing, z = beta * m;
    double loss, d;
    if (a.kind == PairLoss::kSigmoid) {
      loss = (1 - eps) * softplus(-z);
      if (eps > 0) loss += eps * softplus(z);
      d = beta * (1 / (1 + exp(-z)) - (1 - eps));
    } else if (a.kind == PairLoss::kHinge) {
      loss = z < 1 ? 1 - z : (z >= 1 ? 0 : z);  // neither: a NaN, kept
      d = z < 1 ? -beta : (z >= 1 ? 0 : z);
    } else {
      const double off = m - 1 / (2 * beta);
      loss = off * off;
      d = 2 * off;
    }
    a.logps[i] = (float)total[0];
    a.logps[i + P] = (float)total[1];
    a.dseq[i] = (float)(d * a.weight);
    a.dseq[i + P] = (float)(-d * a.weight);
    a.scale[i] = (float)(1 / tokens[0]);
    a.scale[i + P] = (float)(1 / tokens[1]);
    (a.reduced ? a.pair_loss : a.loss)[i] = (float)loss;
  }
  if (!a.reduced || !last_block(a.ticket)) return;
  double v = 0;
  for (int k = threadIdx.x; k < P; k += blockDim.x) v += __ldcg(a.pair_loss + k);
  v = block_sum(v, red);
  if (threadIdx.x == 0) a.loss[0] = (float)(v * a.weight);
}

// exp(d) - 1 - d without the cancellation of small d: below 1/8 the series to d^7 is exact to fp32.
__device__ __forceinline__ float exp_excess(float d) {
  if (fabsf(d) < 0.125f) {
    const float q = 1.f / 2 + d * (1.f / 6 + d * (1.f / 24 + d * (1.f / 120 + d * (1.f / 720 + d * (1.f / 5040)))));
    return d * d * q;
  }
  return expm1f(d) - d;
}

struct TokenTerms {
  float loss, kl, clipped, slope;  // slope: d loss / d logp
};

__device__ __forceinline__ TokenTerms policy_token(const PolicyArgs& a, long long row, long long b, float logp) {
  const float adv = a.adv[a.adv_per_token ? row : b];
  const float r = a.old_logps != nullptr ? expf(logp - a.old_logps[row]) : (logp != logp ? logp : 1.f);
  const float held_r = r < a.clip_lo ? a.clip_lo : (r > a.clip_hi ? a.clip_hi : r);
  const float free = r * adv, held = held_r * adv;
  TokenTerms t;
  t.loss = free <= held ? -free : -held;
  t.slope = free <= held ? -free : (held < free ? 0.f : held);  // neither: a NaN, kept
  t.clipped = held < free ? 1.f : 0.f;
  t.kl = 0.f;
  if (a.ref_logps != nullptr) {
    const float d = a.ref_logps[row] - logp;
    t.kl = exp_excess(d);
    t.loss += a.kl_coef * t.kl;
    t.slope -= a.kl_coef * expm1f(d);
  }
  return t;
}

// One CTA for each sequence: how many of its tokens count. Also clears the ticket.
__global__ void __launch_bounds__(256) policy_count_kernel(PolicyArgs a) {
  __shared__ double red[8];
  const long long base = (long long)blockIdx.x * a.rows.T;
  double n = 0;
  for (int t = threadIdx.x; t < a.rows.T; t += blockDim.x) {
    const int64_t y = a.rows.labels[base + t];
    n += y != a.rows.ignore && y >= 0 && y < a.rows.V;
  }
  n = block_sum(n, red);
  if (threadIdx.x == 0) {
    a.count[blockIdx.x] = (int)n;
    if (blockIdx.x == 0) *a.ticket = 0;
  }
}

// One CTA for each sequence: its tokens' terms, sums and derivatives; the last CTA adds the sequences in order.
__global__ void __launch_bounds__(256) policy_finish_kernel(PolicyArgs a) {
  __shared__ double red[8];
  const int B = gridDim.x, b = blockIdx.x, T = a.rows.T;
  double total = 0;
  for (int k = threadIdx.x; k < B; k += blockDim.x) total += a.count[k];
  total = block_sum(total, red);
  const double mine = a.count[b];
  const double w = a.mean == TokenMean::kTokens      ? 1 / fmax(total, 1.0)
                   : a.mean == TokenMean::kSequences ? 1 / (fmax(mine, 1.0) * B)
                                                     : 1.0;
  const long long base = (long long)b * T;
  double v[3] = {0, 0, 0};
  for (int t = threadIdx.x; t < T; t += blockDim.x) {
    const long long row = base + t;
    const int64_t y = a.rows.labels[row];
    if (y == a.rows.ignore || y < 0 || y >= a.rows.V) {
      a.dtok[row] = 0.f;
      continue;
    }
    const TokenTerms k = policy_token(a, row, b, a.logps[row]);
    a.dtok[row] = (float)(k.slope * w);
    v[0] += k.loss;
    v[1] += k.kl;
    v[2] += k.clipped;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    v[i] = block_sum(v[i], red);
    if (threadIdx.x == 0) a.seq[4 * b + i] = i == 0 ? v[i] * w : v[i];
  }
  if (!last_block(a.ticket)) return;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    double u = 0;
    for (int k = threadIdx.x; k < B; k += blockDim.x) u += __ldcg(a.seq + 4 * k + i);
    u = block_sum(u, red);
    if (threadIdx.x == 0) (i == 0 ? a.loss : i == 1 ? a.kl : a.clipped)[0] = (float)(i == 0 ? u : u / fmax(total, 1.0));
  }
}

template <typename T>
void launch_stats(const LogitRows& r, float* logps, RowStat* stats, unsigned* ticket, cudaStream_t s) {
  const long long rows = (long long)r.B * r.T;
  if (rows == 0) {
    cudaMemsetAsync(ticket, 0, sizeof(unsigned), s);
    return;
  }
  if (r.V > 8192)
    row_stats_kernel<T, 512><<<(unsigned)rows, 512, 0, s>>>(r, logps, stats, ticket);
  else
    row_stats_kernel<T, 128><<<(unsigned)rows, 128, 0, s>>>(r, logps, stats, ticket);
}

template <typename T>
void launch_grad(const LogitGradArgs& a, cudaStream_t s) {
  const long long rows = (long long)a.rows.B * a.rows.T;
  if (rows == 0) return;
  if (a.rows.V > 8192)
    logit_grad_kernel<T, 512><<<(unsigned)rows, 512, 0, s>>>(a);
  else
    logit_grad_kernel<T, 128><<<(unsigned)rows, 128, 0, s>>>(a);
}

void stats_of(const LogitRows& r, float* logps, RowStat* stats, unsigned* ticket, cudaStream_t s) {
  if (r.type == Elem::kBF16)
    launch_stats<__nv_bfloat16>(r, logps, stats, ticket, s);
  else if (r.type == Elem::kF16)
    launch_stats<__half>(r, logps, stats, ticket, s);
  else
    launch_stats<float>(r, logps, stats, ticket, s);
}

}  // namespace

void preference_fwd(const PreferenceArgs& a, cudaStream_t s) {
  stats_of(a.rows, a.logp_tok, a.stats, a.ticket, s);
  preference_finish_kernel<<<a.rows.B / 2, 256, 0, s>>>(a);
}

void policy_fwd(const PolicyArgs& a, cudaStream_t s) {
  stats_of(a.rows, a.logps, a.stats, a.ticket, s);
  policy_count_kernel<<<a.rows.B, 256, 0, s>>>(a);
  policy_finish_kernel<<<a.rows.B, 256, 0, s>>>(a);
}

void logit_grad(const LogitGradArgs& a, cudaStream_t s) {
  if (a.rows.type == Elem::kBF16)
    launch_grad<__nv_bfloat16>(a, s);
  else if (a.rows.type == Elem::kF16)
    launch_grad<__half>(a, s);
  else
    launch_grad<float>(a, s);
}

}  // namespace bw
