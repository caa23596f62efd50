// Preference and policy losses from logits.
//
// Both need log p(y | row) = x_y - lse(x) of the labelled token of every row that counts, and
// both send back coef (onehot(y) - softmax(x)). In base two with c = log2(e) / temperature and
// m = max(x):
//     s = sum_v 2^((x_v - m) c),   log p = (x_y - m) / temperature - ln 2 log2 s,   p_v = 2^((x_v - m) c) / s.
// The maximum is taken off before the scaling: x_v c - m c in one step would overflow where a
// mask put the type's lowest value. Sums are fp32 within a row (each thread its share) and fp64
// over a sequence's tokens and over pairs.
//
// A row whose label is ignored is not read: whatever stands there, its log-probability is 0
// and its gradient is 0.
//
// What bounds them. Long rows: memory. 8 x 1024 x 128256 bf16 logits, a quarter of the rows ignored, on one B200 whose copy
// rate is 6.55 TB/s (launches one by one, the L2 flushed before each):
//     statistics  read 1.58 GB            264 us   6.0 TB/s   (the exponential's unit is 68 % busy beside it)
//     gradient    read 1.58, write 2.10   559 us   6.6 TB/s
//     policy      the same bytes, once    641 us   5.7 TB/s   with its two small kernels
//     gradient under a loss gradient that is not 1: read 1.58, write 1.58 (the ignored rows have their zeros) 510 us
// Passes of a program one behind the other wait for one another's write-backs: 827..852 us for a preference step,
// 644..700 us for a policy step, 1157 us for one whose loss gradient is not 1.
// Short and middle rows: the chain of one row. A warp (or a small CTA) loads a row, takes its maximum, exponentials and
// sums and leaves, with nothing of the next row on its way: 65536 x 1024 statistics 43 us where reading takes 15, with DRAM
// 46 %, issue slots 64 % and the exponential's unit 55 % busy. Rows of 12 to 96 KB take the policy's second read from L2.
// The table above kShort has them all with their floors.
// The preference loss needs both passes over HBM, since a pair's coefficient needs every token of both sequences. The
// policy's does not, and takes them in one kernel.
// Tried and slower for the policy: the row in registers over a cluster of CTAs, joined through distributed shared memory
// (1020 us: a row's chain of load, barrier and store is too long for the few CTAs that fit); persistent CTAs with an
// asynchronous ring across rows (843 us: too few warps for the arithmetic); persistent CTAs that refill the kept part with
// the next row's head during the second pass (767 us). A polynomial on the FMA pipe for a quarter of the exponentials costs more issue slots
// than it frees (statistics 266 -> 288 us).
#include "logit_loss.cuh"

#include "logit_rows.cuh"

namespace bw {
namespace {

template <typename T, int kGroup>
__global__ void __launch_bounds__(Place<kGroup>::kThreads, kGroup == 32 ? 10 : 12)
    row_stats_kernel(LogitRows r, float* __restrict__ logps, RowStat* __restrict__ stats, unsigned* __restrict__ ticket) {
  __shared__ float2 parts[32];
  const long long row = Place<kGroup>::row();
  const int tid = Place<kGroup>::tid();
  if (row == 0 && tid == 0) *ticket = 0;
  if (row >= (long long)r.B * r.T) return;
  const int y = row_label(r, row);
  if (y < 0) {
    if (tid == 0) {
      logps[row] = 0.f;
      stats[row] = RowStat{0.f, 0.f};
    }
    return;
  }
  const T* x = row_ptr<T>(r, row);
  const float c = kLog2e * r.inv_temp;
  float m, s;
  row_stats<T, kGroup>(RowSpan<T>(x, r.V), c, m, s, parts);
  if (tid == 0) {
    const float base = base_of(m);
    logps[row] = label_logp(ElemOf<T>::up(x[y]), base, r.inv_temp, s);
    stats[row] = RowStat{base, 1.f / s};
  }
}

// ---------------------------------------------------------------- gradient
// What the gradient of a row is made of.
struct RowGrad {
  int y;
  float base, c, k, coef;  // k = -coef / s
  bool aligned;            // the gradient's row starts at the same place within 16 bytes
};

// Writes coef (onehot - softmax) of kUnroll vectors.
template <typename T, int kStride>
__device__ __forceinline__ void put(const RowSpan<T>& span, T* out, int j, bool whole, const uint4 (&v)[kUnroll],
                                    const RowGrad& g) {
  constexpr int N = kVecOf<T>;
  if (whole && g.aligned) {
    const int lo = span.first(j);
    uint4* p = reinterpret_cast<uint4*>(out + lo);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      __stcs(p + u * kStride, grad_of<T>(v[u], lo + u * kStride * N, g.y, g.base, g.c, g.k, g.coef));
    return;
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int lo = span.first(j + u * kStride);
    if (lo < span.V) store_vec<T>(out, span.V, lo, grad_of<T>(v[u], lo, g.y, g.base, g.c, g.k, g.coef), g.aligned);
  }
}

template <typename T>
__device__ __forceinline__ RowGrad row_grad_of(const RowSpan<T>& span, const T* out, int y, float base, float inv_s, float c,
                                               float coef) {
  const bool aligned = (int)((reinterpret_cast<uintptr_t>(out) % 16) / sizeof(T)) == span.shift;
  return RowGrad{y, base, c, -coef * inv_s, coef, aligned};
}

// The gradient of a row, read for the last time.
template <typename T, int kGroup>
__device__ __forceinline__ void row_grad(const RowSpan<T>& span, T* out, const RowGrad& g) {
  constexpr int kHold = kGroup * kUnroll;
  const int tid = Place<kGroup>::tid();
  for (int j = tid; j < span.nv; j += kHold) {
    const bool whole = span.inner(j - tid, kHold);
    uint4 v[kUnroll];
    fetch<T, kGroup, true>(span, j, whole, v);
    put<T, kGroup>(span, out, j, whole, v, g);
  }
}

// coef (onehot - softmax) / temperature of a row. A zero coefficient (an ignored row, a clipped token)
// writes zeros without reading the row.
template <typename T, int kGroup>
__device__ __forceinline__ void logit_grad_row(const LogitGradArgs& a, long long row) {
  const LogitRows& r = a.rows;
  const long long b = row / r.T, t = row - b * r.T;
  const int y = row_label(r, row);
  if (y < 0 && a.unit_grad) return;
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
    zero_row<T, kGroup>(out, r.V);
    return;
  }
  const RowStat st = a.stats[row];
  const RowSpan<T> span(row_ptr<T>(r, row), r.V);
  row_grad<T, kGroup>(span, out, row_grad_of(span, out, y, st.m, st.inv_s, kLog2e * r.inv_temp, coef));
}

// Every row. They run backwards: the last ones read before are the likeliest still in L2.
template <typename T, int kGroup>
__global__ void __launch_bounds__(Place<kGroup>::kThreads) logit_grad_kernel(LogitGradArgs a) {
  const long long row = (long long)a.rows.B * a.rows.T - 1 - Place<kGroup>::row();
  if (row >= 0) logit_grad_row<T, kGroup>(a, row);
}

// Where `out` has the gradient for a loss gradient of 1 (a loss that ends the graph) it is done. For any other the rows
// are computed again from the logits: the numbers in `out` are rounded, and what a scaled loss keeps within the range of
// a 16-bit float is gone from them. As many CTAs as are resident, so that they leave at once where there is nothing to do.
template <typename T, int kGroup>
__global__ void __launch_bounds__(Place<kGroup>::kThreads) logit_regrad_kernel(LogitGradArgs a) {
  if (*a.g_loss == 1.f) return;
  const long long by = (long long)gridDim.x * Place<kGroup>::kRows;
  for (long long row = (long long)a.rows.B * a.rows.T - 1 - Place<kGroup>::row(); row >= 0; row -= by)
    logit_grad_row<T, kGroup>(a, row);
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

// What a token brings along, read before it is needed.
struct TokenIn {
  float adv, old_logp, ref_logp;
};

__device__ __forceinline__ TokenIn token_in(const PolicyArgs& a, long long row, long long b) {
  return TokenIn{a.adv[a.adv_per_token ? row : b], a.old_logps != nullptr ? a.old_logps[row] : 0.f,
                 a.ref_logps != nullptr ? a.ref_logps[row] : 0.f};
}

__device__ __forceinline__ TokenTerms policy_token(const PolicyArgs& a, const TokenIn& in, float logp) {
  const float adv = in.adv;
  const float r = a.old_logps != nullptr ? expf(logp - in.old_logp) : (logp != logp ? logp : 1.f);
  const float held_r = r < a.clip_lo ? a.clip_lo : (r > a.clip_hi ? a.clip_hi : r);
  const float free = r * adv, held = held_r * adv;
  TokenTerms t;
  t.loss = free <= held ? -free : -held;
  t.slope = free <= held ? -free : (held < free ? 0.f : held);  // neither: a NaN, kept
  t.clipped = held < free ? 1.f : 0.f;
  t.kl = 0.f;
  if (a.ref_logps != nullptr) {
    const float d = in.ref_logp - logp;
    t.kl = exp_excess(d);
    if (a.kl_coef != 0.f) {  // an infinite distance that is only reported leaves the loss alone
      t.loss += a.kl_coef * t.kl;
      t.slope -= a.kl_coef * expm1f(d);
    }
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

// The sequences' counts in one: with up to kFewSequences every row adds them itself.
constexpr int kFewSequences = 32;

__global__ void __launch_bounds__(1024) policy_total_kernel(PolicyArgs a) {
  __shared__ double red[32];
  double n = 0;
  for (int k = threadIdx.x; k < a.rows.B; k += blockDim.x) n += a.count[k];
  n = block_sum(n, red);
  if (threadIdx.x == 0) a.count[a.rows.B] = (int)n;
}

// A token's share in the loss, from the tokens that count; the same in every lane of a warp.
__device__ __forceinline__ float token_weight(const PolicyArgs& a, long long b) {
  if (a.mean == TokenMean::kSum) return 1.f;
  if (a.mean == TokenMean::kSequences) return 1.f / ((float)max(a.count[b], 1) * a.rows.B);
  int n;
  if (a.rows.B > kFewSequences) {
    n = a.count[a.rows.B];
  } else {
    const int lane = threadIdx.x & 31;
    n = lanes_sum(lane < a.rows.B ? a.count[lane] : 0);
  }
  return 1.f / max(n, 1);
}

// The terms of every token, for calls that take no gradient along.
__global__ void __launch_bounds__(256) policy_token_kernel(PolicyArgs a) {
  const long long b = blockIdx.x, base = b * a.rows.T;
  const float w = token_weight(a, b);
  for (int t = threadIdx.x; t < a.rows.T; t += blockDim.x) {
    const long long row = base + t;
    const int64_t y = a.rows.labels[row];
    TokenTerms k{0.f, 0.f, 0.f, 0.f};
    if (y != a.rows.ignore && y >= 0 && y < a.rows.V) k = policy_token(a, token_in(a, row, b), a.logps[row]);
    a.dtok[row] = k.slope * w;
    a.tok[row] = make_float4(k.loss * w, k.kl, k.clipped, 0.f);
  }
}

// One CTA for each sequence: its tokens' sums; the last CTA adds the sequences in order.
__global__ void __launch_bounds__(256) policy_finish_kernel(PolicyArgs a) {
  __shared__ double red[8];
  const int B = gridDim.x, b = blockIdx.x, T = a.rows.T;
  const long long base = (long long)b * T;
  double v[3] = {0, 0, 0};
  for (int t = threadIdx.x; t < T; t += blockDim.x) {
    const float4 k = a.tok[base + t];
    v[0] += k.x;
    v[1] += k.y;
    v[2] += k.z;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    v[i] = block_sum(v[i], red);
    if (threadIdx.x == 0) a.seq[4 * b + i] = v[i];
  }
  if (!last_block(a.ticket)) return;
  double n = 0;
  for (int k = threadIdx.x; k < B; k += blockDim.x) n += a.count[k];
  n = fmax(block_sum(n, red), 1.0);
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    double u = 0;
    for (int k = threadIdx.x; k < B; k += blockDim.x) u += __ldcg(a.seq + 4 * k + i);
    u = block_sum(u, red);
    if (threadIdx.x == 0) (i == 0 ? a.loss : i == 1 ? a.kl : a.clipped)[0] = (float)(i == 0 ? u : u / n);
  }
}

// ---------------------------------------------------------------- loss and gradient in one kernel
// A token's coefficient needs its own row only, so the group that took a row's statistics writes its gradient at once and
// reads the row a second time: from L2, which holds the few rows that are between their two passes at any time.

// What of a row that counts goes out, from its maximum and sum; the gradient's coefficient, the same in every thread.
__device__ __forceinline__ float policy_out(const PolicyArgs& a, long long row, const TokenIn& in, float w, float xy, float m,
                                            float s, bool first) {
  const float base = base_of(m), logp = label_logp(xy, base, a.rows.inv_temp, s);
  const TokenTerms k = policy_token(a, in, logp);
  if (first) {
    a.logps[row] = logp;
    a.stats[row] = RowStat{base, 1.f / s};
    a.dtok[row] = k.slope * w;
    a.tok[row] = make_float4(k.loss * w, k.kl, k.clipped, 0.f);
  }
  return k.slope * w * a.rows.inv_temp;
}

// The same of a row that does not.
template <typename T, int kGroup>
__device__ __forceinline__ void policy_skip(const PolicyArgs& a, long long row, T* out) {
  if (Place<kGroup>::tid() == 0) {
    a.logps[row] = a.dtok[row] = 0.f;
    a.stats[row] = RowStat{0.f, 0.f};
    a.tok[row] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  zero_row<T, kGroup>(out, a.rows.V);
}

template <typename T>
__device__ __forceinline__ T* grad_row(const PolicyArgs& a, long long row) {
  const long long b = row / a.rows.T;
  return reinterpret_cast<T*>(a.grad) + b * a.gsb + (row - b * a.rows.T) * a.gst;
}

template <typename T, int kGroup, int kMin>
__global__ void __launch_bounds__(Place<kGroup>::kThreads, kMin) policy_row_kernel(PolicyArgs a) {
  __shared__ float2 parts[32];
  const LogitRows& r = a.rows;
  const long long row = Place<kGroup>::row();
  if (row >= (long long)r.B * r.T) return;
  const int y = row_label(r, row);
  T* out = grad_row<T>(a, row);
  if (y < 0) {
    policy_skip<T, kGroup>(a, row, out);
    return;
  }
  const T* x = row_ptr<T>(r, row);
  const RowSpan<T> span(x, r.V);
  const long long b = row / r.T;
  const float c = kLog2e * r.inv_temp, xy = ElemOf<T>::up(x[y]), w = token_weight(a, b);
  const TokenIn in = token_in(a, row, b);
  float m, s;
  row_stats<T, kGroup>(span, c, m, s, parts);
  const float coef = policy_out(a, row, in, w, xy, m, s, Place<kGroup>::tid() == 0);
  if (coef == 0.f)
    zero_row<T, kGroup>(out, r.V);
  else
    row_grad<T, kGroup>(span, out, row_grad_of(span, out, y, base_of(m), 1.f / s, c, coef));
}

// Long rows, two CTAs of an SM: the first kKept vectors are all asked for at once, into shared memory, and stay there for the
// second pass, which asks for the rest again (from L2) three steps ahead as places come free. A thread only reads the places
// it filled itself.
constexpr int kLongThreads = 512, kLongHold = kLongThreads * kUnroll, kKept = 3 * kLongHold;

// The step of vectors from j0 on, on its way to the places of this thread from `to` on; nothing where the row has ended.
template <typename T>
__device__ __forceinline__ void keep_step(uint4* to, const RowSpan<T>& span, int j0) {
  const int j = j0 + (int)threadIdx.x;
  to += threadIdx.x;
  if (span.inner(j0, kLongHold)) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to + u * kLongThreads)),
                   "l"(span.vec(j + u * kLongThreads))
                   : "memory");
  } else if (j0 < span.nv) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) to[u * kLongThreads] = span.template load<false>(j + u * kLongThreads);
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}

template <typename T>
__global__ void __launch_bounds__(kLongThreads, 2) policy_long_kernel(PolicyArgs a) {
  extern __shared__ uint4 keep[];  // [kKept]
  __shared__ float2 parts[32];
  const LogitRows& r = a.rows;
  const long long row = blockIdx.x, b = row / r.T;
  const int tid = threadIdx.x, y = row_label(r, row);
  T* out = grad_row<T>(a, row);
  if (y < 0) {
    policy_skip<T, kLongThreads>(a, row, out);
    return;
  }
  const T* x = row_ptr<T>(r, row);
  const RowSpan<T> span(x, r.V);
  for (int j0 = 0; j0 < kKept; j0 += kLongHold) keep_step<T>(keep + j0, span, j0);
  const float c = kLog2e * r.inv_temp, xy = ElemOf<T>::up(x[y]), w = token_weight(a, b);
  const TokenIn in = token_in(a, row, b);
  uint4 v[kUnroll], ahead[kUnroll];
  const auto load = [&](int j0) {
    fetch<T, kLongThreads, false>(span, j0 + tid, span.inner(j0, kLongHold), ahead);
  };
  load(kKept);
  float m = -INFINITY, s = 0.f;
  const auto kept = [&](int j0) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = keep[j0 + u * kLongThreads + tid];
    take<T>(v, c, m, s);
  };
  asm volatile("cp.async.wait_group 2;" ::: "memory");
  kept(0);
  asm volatile("cp.async.wait_group 1;" ::: "memory");
  kept(kLongHold);
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  kept(2 * kLongHold);
  for (int j0 = kKept; j0 < span.nv; j0 += kLongHold) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = ahead[u];
    if (j0 + kLongHold < span.nv) load(j0 + kLongHold);
    take<T>(v, c, m, s);
  }
  merge_group<kLongThreads>(m, s, c, parts);
  const float coef = policy_out(a, row, in, w, xy, m, s, tid == 0);
  if (coef == 0.f) {
    zero_row<T, kLongThreads>(out, r.V);
    return;
  }
  const RowGrad g = row_grad_of(span, out, y, base_of(m), 1.f / s, c, coef);
  for (int j0 = 0, at = 0; j0 < span.nv; j0 += kLongHold) {
    asm volatile("cp.async.wait_group 2;" ::: "memory");
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = keep[at + u * kLongThreads + tid];
    put<T, kLongThreads>(span, out, j0 + tid, span.inner(j0, kLongHold), v, g);
    keep_step<T>(keep + at, span, j0 + kKept);
    at = at == kKept - kLongHold ? 0 : at + kLongHold;
  }
}

template <int kGroup>
unsigned grid_of(const LogitRows& r) {
  return (unsigned)(((long long)r.B * r.T + Place<kGroup>::kRows - 1) / Place<kGroup>::kRows);
}

// The threads of a row by its vectors of 16 bytes. Short rows want warps (no barrier, four to a CTA), long ones threads
// enough for their loads; measured in us on one B200, bf16 (the fourth fp16), a quarter of the rows ignored, by threads of a
// row, each launch by itself after a flush of the L2, with the loss's own small kernels (about 5 us). Before the bar: what
// reading, or reading and writing, takes at the copy rate (writes of less than the L2's 126 MB need not wait for it):
//     rows x logits   vectors   statistics                gradient                           policy
//     65536 x 1024        128    15 | 32: 43,  128: 106    36 | 32: 37,  128: 86              36 | 32: 80,  128: 213
//     32768 x 4000        500    30 | 32: 59,  128: 70     70 | 32: 68,  128: 76              70 | 32: 111, 128: 147
//     16384 x 16000      2000    60 | 32: 96,  128: 88    140 | 32: 143, 128: 133, 256: 133  140 | 128: 190, 256: 219
//     1998 x 32003       4000    15 | 128: 39, 512: 41     34 | 128: 37, 256: 33,  512: 41    34 | 128: 72, 256: 68
//     8192 x 128256     16032   241 | 128: 264, 512: 266  561 | 256: 569, 512: 557           561 | 256: 813, long: 641
constexpr int kShort = 768;

template <typename T, int kGroup, int kMin>
void policy_rows(const PolicyArgs& a, cudaStream_t s) {
  policy_row_kernel<T, kGroup, kMin><<<grid_of<kGroup>(a.rows), Place<kGroup>::kThreads, 0, s>>>(a);
}

template <typename T>
void rows_of(const PolicyArgs& a, cudaStream_t s) {
  const int n = a.rows.V / kVecOf<T>;
  if (n <= kShort) return policy_rows<T, 32, 8>(a, s);
  if (n <= 3072) return policy_rows<T, 128, 8>(a, s);
  if (n <= kKept) return policy_rows<T, 256, 4>(a, s);
  constexpr int kBytes = kKept * 16;
  cudaFuncSetAttribute(policy_long_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
  policy_long_kernel<T><<<grid_of<kLongThreads>(a.rows), kLongThreads, kBytes, s>>>(a);
}

template <typename T>
void launch_stats(const LogitRows& r, float* logps, RowStat* stats, unsigned* ticket, cudaStream_t s) {
  if (r.V / kVecOf<T> <= kShort)
    row_stats_kernel<T, 32><<<grid_of<32>(r), Place<32>::kThreads, 0, s>>>(r, logps, stats, ticket);
  else
    row_stats_kernel<T, 128><<<grid_of<128>(r), 128, 0, s>>>(r, logps, stats, ticket);
}

template <typename T, int kGroup>
void launch_grad_rows(const LogitGradArgs& a, cudaStream_t s) {
  constexpr int kThreads = Place<kGroup>::kThreads;
  const unsigned all = grid_of<kGroup>(a.rows), resident = 148 * 2048 / kThreads;
  if (a.unit_grad)
    logit_regrad_kernel<T, kGroup><<<all < resident ? all : resident, kThreads, 0, s>>>(a);
  else
    logit_grad_kernel<T, kGroup><<<all, kThreads, 0, s>>>(a);
}

template <typename T>
void launch_grad(const LogitGradArgs& a, cudaStream_t s) {
  const int n = a.rows.V / kVecOf<T>;
  if (n <= kShort) return launch_grad_rows<T, 32>(a, s);
  if (n <= 8192) return launch_grad_rows<T, 256>(a, s);
  launch_grad_rows<T, 512>(a, s);
}

void stats_of(const LogitRows& r, float* logps, RowStat* stats, unsigned* ticket, cudaStream_t s) {
  if ((long long)r.B * r.T == 0)
    cudaMemsetAsync(ticket, 0, sizeof(unsigned), s);
  else if (r.type == Elem::kBF16)
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

int policy_fwd(const PolicyArgs& a, cudaStream_t s) {
  const bool rows = (long long)a.rows.B * a.rows.T > 0;
  if (a.grad == nullptr || !rows) stats_of(a.rows, a.logps, a.stats, a.ticket, s);
  policy_count_kernel<<<a.rows.B, 256, 0, s>>>(a);
  const bool many = a.rows.B > kFewSequences;
  if (many) policy_total_kernel<<<1, 1024, 0, s>>>(a);
  if (a.grad == nullptr || !rows)
    policy_token_kernel<<<a.rows.B, 256, 0, s>>>(a);
  else if (a.rows.type == Elem::kBF16)
    rows_of<__nv_bfloat16>(a, s);
  else if (a.rows.type == Elem::kF16)
    rows_of<__half>(a, s);
  else
    rows_of<float>(a, s);
  policy_finish_kernel<<<a.rows.B, 256, 0, s>>>(a);
  return (a.grad == nullptr ? 4 : 3) + many;
}

void logit_grad(const LogitGradArgs& a, cudaStream_t s) {
  if ((long long)a.rows.B * a.rows.T == 0) return;
  if (a.rows.type == Elem::kBF16)
    launch_grad<__nv_bfloat16>(a, s);
  else if (a.rows.type == Elem::kF16)
    launch_grad<__half>(a, s);
  else
    launch_grad<float>(a, s);
}

}  // namespace bw
