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
// maximum needs anyway), the step that it came in, and the maximum of its other steps. The K-th largest of the threads'
// maxima is a lower bound of the K-th largest logit, so that the K best lie within the elements of the threads that
// reach it: K threads of the row's, plus ties, and of each the one step unless another step reaches it too. A search over the
// bits of the maxima finds the bound; all threads read those steps again (some 2 % of a row; all steps of the K threads were
// 35 % more bytes from memory) and note the elements that reach it, hardly more than K; each of those is ranked by counting the
// larger ones. Where ties make steps or elements more than is noted, all elements of the threads are read, and one warp
// takes them into a sorted list with an entry for each lane.
//
// A row whose label is ignored is not read. A NaN in a row makes its numbers NaN; among the alternatives it is the
// largest.
#include "token_scores.cuh"

#include "logit_rows.cuh"

namespace bw {
namespace {

using bf16 = __nv_bfloat16;

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

// Words of elements no smaller than `low`; a NaN stays.
__device__ __forceinline__ uint32_t word_floor(uint32_t a, uint32_t low, bf16) {
  const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&low));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t word_floor(uint32_t a, uint32_t low, __half) {
  const __half2 m = __hmax2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&low));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t word_floor(uint32_t a, uint32_t low, float) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(__uint_as_float(a)), "f"(__uint_as_float(low)));
  return __float_as_uint(m);
}

// The word that elements are raised to before t is taken: 250 / c or more below the base, where 2^t is 0 and t still a number.
// Rounded down, so that no element that counts is raised. -inf, which raises none, where the type's range ends before.
__device__ __forceinline__ uint32_t floor_of(float base, float reach, bf16) {
  const bf16 f = __float2bfloat16_rd(__fsub_rd(base, reach));
  const __nv_bfloat162 two = __halves2bfloat162(f, f);
  return *reinterpret_cast<const uint32_t*>(&two);
}
__device__ __forceinline__ uint32_t floor_of(float base, float reach, __half) {
  const __half f = __float2half_rd(__fsub_rd(base, reach));
  const __half2 two = __halves2half2(f, f);
  return *reinterpret_cast<const uint32_t*>(&two);
}
__device__ __forceinline__ uint32_t floor_of(float base, float reach, float) {
  return __float_as_uint(__fsub_rd(base, reach));
}

// kRaise: by `low`. Otherwise, at the lower end of the type's range, t itself is held to what counts.
template <typename T, bool kRaise, int K>
__device__ __forceinline__ void add_scores(const uint4 (&v)[K], float c, float base, uint32_t low, Sums& a) {
  const float2 off = make_float2(-base, -base), cc = make_float2(c, c);
  float2 s = make_float2(0.f, 0.f), w = make_float2(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float f[kVecOf<T>];
    uint4 r = v[k];
    if (kRaise)
      r = make_uint4(word_floor(r.x, low, T()), word_floor(r.y, low, T()), word_floor(r.z, low, T()), word_floor(r.w, low, T()));
    raw_up<T>(r, f);
#pragma unroll
    for (int i = 0; i < kVecOf<T> / 2; ++i) {
      float2 t = __fmul2_rn(__fadd2_rn(make_float2(f[2 * i], f[2 * i + 1]), off), cc);
      const float2 e = make_float2(ex2(t.x), ex2(t.y));
      s = __fadd2_rn(s, e);
      if (!kRaise) t = make_float2(fmaxf(t.x, kFar), fmaxf(t.y, kFar));
      w = __ffma2_rn(e, t, w);
    }
  }
  a.s += s.x + s.y;
  a.w += w.x + w.y;
}

template <typename T, int K>
__device__ __forceinline__ void take_scores(const uint4 (&v)[K], float c, float reach, float top, Sums& a) {
  if (top > a.m) {
    rebase(a, top, c);
    a.m = top;
  }
  const float base = base_of(a.m);
  const uint32_t low = floor_of(base, reach, T());
  if ((sizeof(T) == 2 ? low & 0xffffu : low) != ElemOf<T>::kNegInf) add_scores<T, true>(v, c, base, low, a);
  else add_scores<T, false>(v, c, base, low, a);
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

constexpr int kNoted = 96, kSteps = 256;  // elements of a row that reach the bound, and steps that have them, for the quick way

template <int kGroup>
struct ScoreShared {
  static constexpr int kWarps = kGroup / 32;
  Sums parts[kWarps];
  int owners[kGroup];  // the threads whose maxima reach the bound
  int steps[kSteps];   // their steps that do: thread + step * kGroup
  int count[3];        // of the owners, of the elements noted, of the steps
  unsigned long long noted[kNoted];
};

template <int kGroup>
__device__ __forceinline__ void group_sync() {
  if (kGroup > 32) __syncthreads();
  else __syncwarp();
}

template <int kGroup>
__device__ __forceinline__ int group_count(bool x) {
  return kGroup > 32 ? __syncthreads_count(x) : __popc(__ballot_sync(0xffffffffu, x));
}

// The maximum of a thread's elements, the step it came in, and the maximum of its other steps.
struct Best {
  float most = -INFINITY, other = -INFINITY;
  int step = 0;
  __device__ __forceinline__ void take(float top, int at) {
    if (top > most) {
      other = most;
      most = top;
      step = at;
    } else {
      other = fmaxf(other, top);
    }
  }
};

// The row's alternatives. `mine`: of the calling thread's vectors (tid, tid + kGroup, ...), kUnroll of them a step.
template <typename T, int kGroup>
__device__ __forceinline__ void alternatives(const ScoreArgs& a, const RowSpan<T>& span, long long row, const Best& mine, bool has_nan,
                                             float base, float log2_s, ScoreShared<kGroup>& sh) {
  constexpr int N = kVecOf<T>;
  const int tid = Place<kGroup>::tid(), lane = threadIdx.x & 31, K = a.top;
  // The largest number with 16 significant bits that K maxima reach, bit by bit. Small rows and rows with a NaN, which the
  // maxima pass over, are looked at whole.
  const uint32_t key = (uint32_t)(key_of(mine.most, 0) >> 32);
  uint32_t bound = 0;
  if (!has_nan) {
#pragma unroll 1
    for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1)
      if (group_count<kGroup>(key >= (bound | bit)) >= K) bound |= bit;
  }
  const bool owner = has_nan || key >= bound;
  if (tid < 3) sh.count[tid] = 0;
  group_sync<kGroup>();
  constexpr int kHold = kGroup * kUnroll;
  const int all_steps = (span.nv + kHold - 1) / kHold;
  if (owner) {
    sh.owners[atomicAdd(&sh.count[0], 1)] = tid;
    const bool more = has_nan || (uint32_t)(key_of(mine.other, 0) >> 32) >= bound;
    const int n = more ? all_steps : 1, at = atomicAdd(&sh.count[2], n);
    for (int i = 0; i < n && at + i < kSteps; ++i) sh.steps[at + i] = tid + (more ? i : mine.step) * kGroup;
  }
  group_sync<kGroup>();
  const bool few = sh.count[2] <= kSteps;
  const int owners = sh.count[0], per = all_steps * kUnroll;
  for (int u = tid; few && u < sh.count[2] * kUnroll; u += kGroup) {
    const int unit = sh.steps[u / kUnroll], j = unit % kGroup + unit / kGroup * kHold + u % kUnroll * kGroup, lo = span.first(j);
    if (j >= span.nv) continue;
    float f[N];
    raw_up<T>(span.template load<false>(j), f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const unsigned long long x = key_of(f[i], lo + i);
      if ((uint32_t)(x >> 32) >= bound && lo + i >= 0 && lo + i < span.V) {
        const int at = atomicAdd(&sh.count[1], 1);
        if (at < kNoted) sh.noted[at] = x;
      }
    }
  }
  group_sync<kGroup>();
  const int found = sh.count[1];
  if (few && found <= kNoted) {
    for (int i = tid; i < found; i += kGroup) {
      const unsigned long long x = sh.noted[i];
      int rank = 0;
      for (int o = 0; o < found; ++o) rank += sh.noted[o] > x;
      if (rank < K) {
        a.top_ids[row * K + rank] = (int)~(uint32_t)x;
        a.top_logps[row * K + rank] = label_logp_of(value_of(x), base, a.rows.inv_temp, log2_s);
      }
    }
    return;
  }
  if (tid >= 32) return;
  unsigned long long list = 0, last = bound ? ((unsigned long long)bound << 32) - 1 : 0;
  for (int u0 = 0; u0 < owners * per; u0 += 32) {
    const int u = u0 + lane, j = u < owners * per ? sh.owners[u / per] + u % per * kGroup : span.nv, lo = span.first(j);
    float f[N];
    raw_up<T>(span.template load<false>(j), f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool in = j < span.nv && lo + i >= 0 && lo + i < span.V;
      insert(in ? key_of(f[i], lo + i) : 0ull, K, list, last);
    }
  }
  if (lane < K) {
    a.top_ids[row * K + lane] = (int)~(uint32_t)list;
    a.top_logps[row * K + lane] = label_logp_of(value_of(list), base, a.rows.inv_temp, log2_s);
  }
}

template <typename T, int kGroup, bool kTop>
__global__ void __launch_bounds__(Place<kGroup>::kThreads, kGroup == 32 ? 10 : 1536 / kGroup) scores_kernel(ScoreArgs a) {
  __shared__ ScoreShared<kGroup> shared[kTop ? Place<kGroup>::kRows : 1];
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
  const float c = kLog2e * r.inv_temp, reach = 250.f / c;
  Sums sum{-INFINITY, 0.f, 0.f};
  Best mine;
  for (int j = tid; j < span.nv; j += kHold) {
    uint4 v[kUnroll];
    fetch<T, kGroup, false>(span, j, span.inner(j - tid, kHold), v);
    const float top = max_of<T>(v);
    take_scores<T>(v, c, reach, top, sum);
    if constexpr (kTop) mine.take(top, j / kHold);
  }
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
  // A warp to a row while it is short, or while there are rows for all warps: 2^28 bf16 logits in rows of 6,144 take 101 us with a
  // warp and 202 with 256 threads, in rows of 12,288 100 and 163, of 16,384 101 and 127 (with 20 alternatives 198 and 388, 188
  // and 252, 212 and 191); 4,736 rows of 12,288 34 and 44. Of few rows, each is a chain by itself, an eighth as long with 256 threads.
  const int n = a.rows.V / kVecOf<T>;
  if (n <= 768 || (n <= 1536 && (long long)a.rows.B * a.rows.T >= 148 * 32)) return fwd<T, 32>(a, s);
  fwd<T, 256>(a, s);
}

template <typename T, int kGroup>
void bwd(const ScoreGradArgs& a, cudaStream_t s) {
  scores_grad_kernel<T, kGroup><<<grid_of<kGroup>(a.rows), Place<kGroup>::kThreads, 0, s>>>(a);
}

template <typename T>
void bwd_of(const ScoreGradArgs& a, cudaStream_t s) {
  // 2^28 bf16 logits in rows of 4,096: 208 us with a warp to a row and 311 with 256 threads, of 8,192 212 and 202; of 65,536 218
  // with 256 and 205 with 512.
  const int n = a.rows.V / kVecOf<T>;
  if (n <= 768) return bwd<T, 32>(a, s);
  if (n <= 2048) return bwd<T, 256>(a, s);
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
