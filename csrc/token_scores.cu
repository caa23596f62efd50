// Scores of tokens from logits: for every row that counts, with c = log2(e) / temperature, m = max(x),
// t_v = (x_v - m) c, s = sum 2^t_v and w = sum 2^t_v t_v,
//     log p(y) = (x_y - m) / temperature - ln 2 log2 s,     H = ln 2 (log2 s - w / s),
// and the K largest logits with their log-probabilities, the lowest index first among equals. One pass: a new maximum
// multiplies s and w by 2^t0 and adds t0 s to w, t0 being the step of the maximum.
//
// The gradient of a loss with d loss / d log p(y) = a and d loss / d H = b is
//     (a onehot(y) - p_v (a + b (log p_v + H))) / temperature = onehot + 2^t_v (k0 + k1 t_v),
// one fused multiply-add more than that of a softmax.
//
// Alternatives. In the pass each thread only keeps the maximum of its own elements (packed maxima, which the running
// maximum needs anyway). The K-th largest of these maxima is a lower bound of the K-th largest logit, so that the K
// best lie within the elements of the threads that reach it: K threads of the row's, plus ties. Warps read those
// elements again, from the L2 for the most part, and keep a sorted list with one entry for each lane; one warp merges the lists.
//
// A row whose label is ignored is not read. A NaN in a row makes its numbers NaN; among the alternatives it is the
// largest.
#include "token_scores.cuh"

#include "logit_rows.cuh"

namespace bw {
namespace {

// t below this adds nothing to s or w: 2^-200 is 0. It stands for -inf, which would make a NaN of 0 t.
constexpr float kFar = -200.f;

struct Sums {
  float m, s, w;
};

__device__ __forceinline__ void rebase(Sums& a, float to, float c) {
  if (a.m == -INFINITY) return;  // s and w are 0, or a NaN
  const float t0 = fmaxf((a.m - to) * c, kFar), f = ex2(t0);
  a.w = f * fmaf(t0, a.s, a.w);
  a.s *= f;
}

template <typename T, int K>
__device__ __forceinline__ void take_scores(const uint4 (&v)[K], float c, float top, Sums& a) {
  if (top > a.m) {
    rebase(a, top, c);
    a.m = top;
  }
  const float base = base_of(a.m);
  const float2 off = make_float2(-base, -base), cc = make_float2(c, c);
  float2 s = make_float2(0.f, 0.f), w = make_float2(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float f[kVecOf<T>];
    raw_up<T>(v[k], f);
#pragma unroll
    for (int i = 0; i < kVecOf<T> / 2; ++i) {
      const float2 t = __fmul2_rn(__fadd2_rn(make_float2(f[2 * i], f[2 * i + 1]), off), cc);
      const float2 e = make_float2(ex2(t.x), ex2(t.y));
      s = __fadd2_rn(s, e);
      w = __ffma2_rn(e, make_float2(fmaxf(t.x, kFar), fmaxf(t.y, kFar)), w);
    }
  }
  a.s += s.x + s.y;
  a.w += w.x + w.y;
}

__device__ __forceinline__ void merge_lanes(Sums& a, float c) {
  float M = a.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  rebase(a, M, c);
  a.m = M;
  a.s = lanes_sum(a.s);
  a.w = lanes_sum(a.w);
}

// A logit's place in the order: larger first, the lower index among equals, NaN before all.
__device__ __forceinline__ unsigned long long key_of(float x, int index) {
  uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);  // -0 and 0 are equal
  b = x != x ? 0xffffffffu : (b & 0x80000000u ? ~b : b | 0x80000000u);
  return (unsigned long long)b << 32 | (uint32_t)~index;
}

__device__ __forceinline__ float value_of(unsigned long long key) {
  const uint32_t b = (uint32_t)(key >> 32);
  if (b == 0xffffffffu) return NAN;
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

// Puts the lanes' keys (0: none) into the warp's list, lane i holding the i-th largest. `last` is the K-th.
__device__ __forceinline__ void insert(unsigned long long key, int K, unsigned long long& list, unsigned long long& last) {
  const int lane = threadIdx.x & 31;
  unsigned todo = __ballot_sync(0xffffffffu, key > last);
  while (todo) {
    const int from = __ffs(todo) - 1;
    todo &= todo - 1;
    const unsigned long long x = __shfl_sync(0xffffffffu, key, from);
    if (x <= last) continue;
    const unsigned long long before = __shfl_up_sync(0xffffffffu, list, 1);
    if (list < x) list = lane == 0 || before >= x ? x : before;
    const unsigned long long kth = __shfl_sync(0xffffffffu, list, K - 1);  // 0 until the list has K entries
    if (kth > last) last = kth;
  }
}

template <int kGroup>
struct ScoreShared {
  static constexpr int kWarps = kGroup / 32;
  Sums parts[kWarps];
  alignas(16) float tops[kGroup];
  float bound;
  unsigned long long lists[kWarps][32];
};

// The row's alternatives. `mine`: the maximum of the calling thread's vectors (tid, tid + kGroup, ...).
template <typename T, int kGroup>
__device__ __forceinline__ void alternatives(const ScoreArgs& a, const RowSpan<T>& span, long long row, float mine, bool has_nan,
                                             float base, float log2_s, ScoreShared<kGroup>& sh) {
  constexpr int kW = kGroup / 32, N = kVecOf<T>;
  const int tid = Place<kGroup>::tid(), lane = threadIdx.x & 31, warp = kW > 1 ? threadIdx.x >> 5 : 0, K = a.top;
  float bound = -INFINITY;
  if constexpr (kW == 1) {
    int above = 0, equal = 0;
#pragma unroll
    for (int o = 0; o < 32; ++o) {
      const float x = __shfl_sync(0xffffffffu, mine, o);
      above += x > mine;
      equal += x >= mine;
    }
    const unsigned at = __ballot_sync(0xffffffffu, above < K && equal >= K);
    if (at && !has_nan) bound = __shfl_sync(0xffffffffu, mine, __ffs(at) - 1);
  } else {
    sh.tops[tid] = mine;
    if (tid == 0) sh.bound = -INFINITY;
    __syncthreads();
    int above = 0, equal = 0;
    const float4* tops = reinterpret_cast<const float4*>(sh.tops);
#pragma unroll 4
    for (int o = 0; o < kGroup / 4; ++o) {
      const float4 x = tops[o];
      above += (x.x > mine) + (x.y > mine) + (x.z > mine) + (x.w > mine);
      equal += (x.x >= mine) + (x.y >= mine) + (x.z >= mine) + (x.w >= mine);
    }
    if (above < K && equal >= K && !has_nan) sh.bound = mine;  // the same value from each that writes
    __syncthreads();
    bound = sh.bound;
  }
  // The keys that count lie above `last`: at first all whose value is the bound at least.
  unsigned long long list = 0, last = key_of(bound, 0) >> 32 << 32;
  if (last) --last;
  const auto scan = [&](int owner) {
    for (int j0 = owner; j0 < span.nv; j0 += 32 * kGroup) {
      const int j = j0 + lane * kGroup, lo = span.first(j);
      float f[N];
      raw_up<T>(span.template load<false>(j), f);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool in = j < span.nv && lo + i >= 0 && lo + i < span.V;
        insert(in ? key_of(f[i], lo + i) : 0ull, K, list, last);
      }
    }
  };
  if constexpr (kW == 1) {
    unsigned todo = __ballot_sync(0xffffffffu, mine >= bound);
    while (todo) {
      scan(__ffs(todo) - 1);
      todo &= todo - 1;
    }
  } else {
    // The warps share the threads that reach the bound: each takes every kW-th of them.
    int seen = 0;
    for (int w = 0; w < kW; ++w) {
      unsigned todo = __ballot_sync(0xffffffffu, sh.tops[w * 32 + lane] >= bound);
      while (todo) {
        if (seen++ % kW == warp) scan(w * 32 + __ffs(todo) - 1);
        todo &= todo - 1;
      }
    }
    sh.lists[warp][lane] = list;
    __syncthreads();
    if (warp > 0) return;
    for (int w = 1; w < kW; ++w) insert(sh.lists[w][lane], K, list, last);
  }
  if (lane < K) {
    a.top_ids[row * K + lane] = (int)~(uint32_t)list;
    a.top_logps[row * K + lane] = label_logp_of(value_of(list), base, a.rows.inv_temp, log2_s);
  }
}

template <typename T, int kGroup, bool kTop>
__global__ void __launch_bounds__(Place<kGroup>::kThreads) scores_kernel(ScoreArgs a) {
  __shared__ ScoreShared<kGroup> shared[kTop || kGroup > 32 ? Place<kGroup>::kRows : 1];
  constexpr int kW = kGroup / 32, kHold = kGroup * kUnroll;
  const LogitRows& r = a.rows;
  const long long row = Place<kGroup>::row();
  const int tid = Place<kGroup>::tid();
  if (row >= (long long)r.B * r.T) return;
  ScoreShared<kGroup>& sh = shared[kW == 1 && kTop ? threadIdx.x >> 5 : 0];
  const int y = row_label(r, row);
  if (y < 0) {
    if (tid == 0) {
      a.logps[row] = 0.f;
      a.entropy[row] = 0.f;
      if (a.stats != nullptr) a.stats[row] = ScoreStat{0.f, 0.f, 0.f};
    }
    if (kTop)
      for (int i = tid; i < a.top; i += kGroup) {
        a.top_ids[row * a.top + i] = -1;
        a.top_logps[row * a.top + i] = 0.f;
      }
    return;
  }
  const T* x = row_ptr<T>(r, row);
  const RowSpan<T> span(x, r.V);
  const float c = kLog2e * r.inv_temp;
  Sums sum{-INFINITY, 0.f, 0.f};
  for (int j = tid; j < span.nv; j += kHold) {
    uint4 v[kUnroll];
    fetch<T, kGroup, false>(span, j, span.inner(j - tid, kHold), v);
    take_scores<T>(v, c, max_of<T>(v), sum);
  }
  const float mine = sum.m;
  merge_lanes(sum, c);
  if constexpr (kW > 1) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) sh.parts[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = lane < kW ? sh.parts[lane] : Sums{-INFINITY, 0.f, 0.f};
    merge_lanes(sum, c);
  }
  const float base = base_of(sum.m), log2_s = log2f(sum.s);
  if (tid == 0) {
    const float entropy = kLn2 * (log2_s - sum.w / sum.s);
    a.logps[row] = label_logp_of(ElemOf<T>::up(x[y]), base, r.inv_temp, log2_s);
    a.entropy[row] = entropy;
    if (a.stats != nullptr) a.stats[row] = ScoreStat{base, log2_s, entropy};
  }
  if constexpr (kTop) alternatives<T, kGroup>(a, span, row, mine, sum.s != sum.s, base, log2_s, sh);
}

// ---------------------------------------------------------------- gradient
template <typename T, int kGroup>
__global__ void __launch_bounds__(Place<kGroup>::kThreads) scores_grad_kernel(ScoreGradArgs a) {
  constexpr int N = kVecOf<T>, kHold = kGroup * kUnroll;
  const LogitRows& r = a.rows;
  const long long row = (long long)r.B * r.T - 1 - Place<kGroup>::row();  // the last ones read before are the likeliest in L2
  if (row < 0) return;
  const int tid = Place<kGroup>::tid();
  const long long b = row / r.T, t = row - b * r.T;
  T* out = reinterpret_cast<T*>(a.out) + b * a.osb + t * a.ost;
  const int y = row_label(r, row);
  const float ga = y >= 0 && a.g_logps != nullptr ? a.g_logps[row] * r.inv_temp : 0.f;
  const float gb = y >= 0 && a.g_entropy != nullptr ? a.g_entropy[row] * r.inv_temp : 0.f;
  if (ga == 0.f && gb == 0.f) {
    zero_row<T, kGroup>(out, r.V);
    return;
  }
  const ScoreStat st = a.stats[row];
  const RowSpan<T> span(row_ptr<T>(r, row), r.V);
  const float c = kLog2e * r.inv_temp;
  // 2^t p0 is the probability: its factor joins the exponent.
  const float k0 = -(ga + gb * (st.entropy - kLn2 * st.log2_s)), k1 = -gb * kLn2;
  const bool aligned = (int)((reinterpret_cast<uintptr_t>(out) % 16) / sizeof(T)) == span.shift;
  const float2 off = make_float2(-st.base, -st.base), cc = make_float2(c, c), ls = make_float2(-st.log2_s, -st.log2_s);
  for (int j = tid; j < span.nv; j += kHold) {
    const bool whole = span.inner(j - tid, kHold);
    uint4 v[kUnroll];
    fetch<T, kGroup, true>(span, j, whole, v);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int lo = span.first(j + u * kGroup);
      float f[N];
      raw_up<T>(v[u], f);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float2 q = __fmul2_rn(__fadd2_rn(make_float2(f[2 * i], f[2 * i + 1]), off), cc), p = __fadd2_rn(q, ls);
        const float2 e = make_float2(ex2(p.x), ex2(p.y));
        const float2 g = __fmul2_rn(e, __ffma2_rn(make_float2(fmaxf(q.x, kFar), fmaxf(q.y, kFar)), make_float2(k1, k1), make_float2(k0, k0)));
        f[2 * i] = g.x;
        f[2 * i + 1] = g.y;
      }
      if ((unsigned)(y - lo) < (unsigned)N) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (lo + i == y) f[i] += ga;
      }
      const uint4 d = raw_down<T, uint4>(f);
      if (whole && aligned) __stcs(reinterpret_cast<uint4*>(out + lo), d);
      else if (lo < span.V) store_vec<T>(out, span.V, lo, d, aligned);
    }
  }
}

template <int kGroup>
unsigned grid_of(const LogitRows& r) {
  return (unsigned)(((long long)r.B * r.T + Place<kGroup>::kRows - 1) / Place<kGroup>::kRows);
}

template <typename T, int kGroup>
void fwd(const ScoreArgs& a, cudaStream_t s) {
  if (a.top > 0) scores_kernel<T, kGroup, true><<<grid_of<kGroup>(a.rows), Place<kGroup>::kThreads, 0, s>>>(a);
  else scores_kernel<T, kGroup, false><<<grid_of<kGroup>(a.rows), Place<kGroup>::kThreads, 0, s>>>(a);
}

template <typename T>
void fwd_of(const ScoreArgs& a, cudaStream_t s) {
  if (a.rows.V / kVecOf<T> <= 768) return fwd<T, 32>(a, s);
  fwd<T, 256>(a, s);
}

template <typename T, int kGroup>
void bwd(const ScoreGradArgs& a, cudaStream_t s) {
  scores_grad_kernel<T, kGroup><<<grid_of<kGroup>(a.rows), Place<kGroup>::kThreads, 0, s>>>(a);
}

template <typename T>
void bwd_of(const ScoreGradArgs& a, cudaStream_t s) {
  const int n = a.rows.V / kVecOf<T>;
  if (n <= 768) return bwd<T, 32>(a, s);
  if (n <= 8192) return bwd<T, 256>(a, s);
  bwd<T, 512>(a, s);
}

}  // namespace

void token_scores_fwd(const ScoreArgs& a, cudaStream_t s) {
  if ((long long)a.rows.B * a.rows.T == 0) return;
  if (a.rows.type == Elem::kBF16) fwd_of<__nv_bfloat16>(a, s);
  else if (a.rows.type == Elem::kF16) fwd_of<__half>(a, s);
  else fwd_of<float>(a, s);
}

void token_scores_bwd(const ScoreGradArgs& a, cudaStream_t s) {
  if ((long long)a.rows.B * a.rows.T == 0) return;
  if (a.rows.type == Elem::kBF16) bwd_of<__nv_bfloat16>(a, s);
  else if (a.rows.type == Elem::kF16) bwd_of<__half>(a, s);
  else bwd_of<float>(a, s);
}

}  // namespace bw
