// Balance loss of an expert router, forward and backward.
//
// With p = softmax(x) of the N tokens that count, f_e the choices of expert e per token and
// P_e the mean of p_e:
//     loss = E sum_e f_e P_e + z mean(lse^2)
//     dx_ne = g [ E p_ne (f_e - sum_j f_j p_nj) + 2 z lse_n p_ne ] / N        (f is a constant)
// The probabilities add up to one, so any constant may be taken off f: with K / E, its mean, the difference keeps its
// digits where the experts are used nearly alike, and is 0 where they are.
// p is computed again in the backward: writing it would cost as much as reading the logits.
//
// 16 groups of 65536 tokens, 64 experts, top 8, on one B200 (copy rate 6.55 TB/s), us, with the floor of reading (and
// writing) in brackets:
//     forward   bf16 97 + 7 for the joining of the CTAs' sums (20)   fp32 126 + 7 (41)
//     backward  bf16 58 (41)                                         fp32 88 (82)
// The forward is bound by the min / max instructions of the selection (ALU 72 % busy, DRAM 17 %), two thirds of whose merges
// another lane of the token does too. 3 to 7 choices run the network of 8, without the short last merge: top 4 106 us where
// top 8 takes 102 and top 2 77. Where the choices are given there is no selection. The backward takes maximum and sum again,
// which fills its issue slots (74 %).
#include "router_balance.cuh"

#include <cmath>
#include <type_traits>

#include "tc_common.cuh"

namespace bw {
namespace {

constexpr int kWarps = 8;

// Order-preserving key: larger values first, a NaN as infinity, -0 equal to 0. 0 is left for "taken".
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(fminf(v, INFINITY) + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// ---------------------------------------------------------------- up to 256 experts, 8 choices
// 2^log lanes share a token, lane l holds its experts 8 l .. 8 l + 7, and two tokens at once (A, B), whose logits of
// one expert go through the selection side by side: in the halves of a word for 16-bit types. The K-th largest is found by
// sorting each lane's 8 and merging sorted lists over the lanes; then each lane counts its own experts at or above it.
// K rounds of "the largest that is left" took 5 times as long in the kernels below: each round waits for the lanes' maximum.
// Sums and counts stay in registers until a CTA is done, and CTAs leave theirs in a row of a table that one more kernel
// adds in order: no floating atomics, the same result each time.
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The logits of one expert for tokens A and B. A NaN takes part in the selection as infinity.
template <typename T>
struct Pair {
  uint32_t w;
};
template <>
struct Pair<float> {
  float a, b;
};

__device__ __forceinline__ __nv_bfloat162 h2(uint32_t w, __nv_bfloat16) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
__device__ __forceinline__ __half2 h2(uint32_t w, __half) { return *reinterpret_cast<const __half2*>(&w); }
template <typename H>
__device__ __forceinline__ uint32_t word(H h) {
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ Pair<T> larger(Pair<T> x, Pair<T> y) {
  if constexpr (sizeof(T) == 2)
    return Pair<T>{word(__hmax2(h2(x.w, T()), h2(y.w, T())))};
  else
    return Pair<T>{fmaxf(x.a, y.a), fmaxf(x.b, y.b)};
}
template <typename T>
__device__ __forceinline__ Pair<T> smaller(Pair<T> x, Pair<T> y) {
  if constexpr (sizeof(T) == 2)
    return Pair<T>{word(__hmin2(h2(x.w, T()), h2(y.w, T())))};
  else
    return Pair<T>{fminf(x.a, y.a), fminf(x.b, y.b)};
}
// 1 in the low half where A's x >= y, 1 in the high half for B.
template <typename T>
__device__ __forceinline__ uint32_t at_least(Pair<T> x, Pair<T> y) {
  if constexpr (sizeof(T) == 2)
    return __hge2_mask(h2(x.w, T()), h2(y.w, T())) & 0x00010001u;
  else
    return (x.a >= y.a ? 1u : 0u) | (x.b >= y.b ? 0x10000u : 0u);
}
template <typename T>
__device__ __forceinline__ uint32_t alike(Pair<T> x, Pair<T> y) {
  if constexpr (sizeof(T) == 2)
    return __heq2_mask(h2(x.w, T()), h2(y.w, T())) & 0x00010001u;
  else
    return (x.a == y.a ? 1u : 0u) | (x.b == y.b ? 0x10000u : 0u);
}
template <typename T>
__device__ __forceinline__ Pair<T> from_lane(Pair<T> x, int o) {
  if constexpr (sizeof(T) == 2)
    return Pair<T>{__shfl_xor_sync(0xffffffffu, x.w, o)};
  else
    return Pair<T>{__shfl_xor_sync(0xffffffffu, x.a, o), __shfl_xor_sync(0xffffffffu, x.b, o)};
}
template <typename T>
__device__ __forceinline__ float2 both(Pair<T> x) {
  if constexpr (sizeof(T) == 2) {
    float f[2];
    word_up(x.w, f, T());
    return make_float2(f[0], f[1]);
  } else {
    return make_float2(x.a, x.b);
  }
}

template <typename T>
__device__ __forceinline__ void order(Pair<T>& x, Pair<T>& y) {  // the larger first
  const Pair<T> l = larger(x, y);
  y = smaller(x, y);
  x = l;
}

// Batcher's odd-even merge sort of 8, largest first.
template <typename T>
__device__ __forceinline__ void sort8(Pair<T> (&v)[8]) {
  order(v[0], v[1]), order(v[2], v[3]), order(v[4], v[5]), order(v[6], v[7]);
  order(v[0], v[2]), order(v[1], v[3]), order(v[4], v[6]), order(v[5], v[7]);
  order(v[1], v[2]), order(v[5], v[6]);
  order(v[0], v[4]), order(v[1], v[5]), order(v[2], v[6]), order(v[3], v[7]);
  order(v[2], v[4]), order(v[3], v[5]);
  order(v[1], v[2]), order(v[3], v[4]), order(v[5], v[6]);
}

// The kTop largest of two sorted lists, the other one from the lane o away: a bitonic list, sorted again.
template <typename T, int kTop>
__device__ __forceinline__ void merge_top(Pair<T> (&v)[8], int o) {
  Pair<T> other[kTop];
#pragma unroll
  for (int i = 0; i < kTop; ++i) other[i] = from_lane(v[i], o);
#pragma unroll
  for (int i = 0; i < kTop; ++i) v[i] = larger(v[i], other[kTop - 1 - i]);
#pragma unroll
  for (int gap = kTop / 2; gap > 0; gap /= 2)
#pragma unroll
    for (int i = 0; i < kTop; ++i)
      if ((i & gap) == 0) order(v[i], v[i + gap]);
}

// A token's 8 logits of this lane as loaded; experts from E on are -inf.
template <typename T>
struct Raw8 {
  static constexpr int kWords = 2 * (int)sizeof(T);
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const T* x, int e, int E, int vec) {
    constexpr uint32_t kFill = sizeof(T) == 2 ? ElemOf<T>::kNegInf * 0x10001u : ElemOf<T>::kNegInf;
    if (vec == 8) {
#pragma unroll
      for (int k = 0; k < kWords; k += 4) {
        uint4 r = make_uint4(kFill, kFill, kFill, kFill);
        if (e < E) r = __ldg(reinterpret_cast<const uint4*>(x + e) + k / 4);
        words_of(r, w + k);
      }
    } else if (vec == 4) {
      using Half = std::conditional_t<sizeof(T) == 2, uint2, uint4>;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (e + 4 * k < E) {
          words_of(__ldg(reinterpret_cast<const Half*>(x + e + 4 * k)), w + k * kWords / 2);
        } else {
#pragma unroll
          for (int i = 0; i < kWords / 2; ++i) w[k * kWords / 2 + i] = kFill;
        }
      }
    } else {
      float f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = e + k < E ? ElemOf<T>::up(x[e + k]) : -INFINITY;
#pragma unroll
      for (int k = 0; k < kWords; ++k) w[k] = word_down(f + k * 8 / kWords, T());
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int k = 0; k < kWords; ++k) w[k] = 0;
  }
  __device__ __forceinline__ void up(float (&f)[8]) const {
#pragma unroll
    for (int k = 0; k < kWords; ++k) word_up(w[k], f + k * 8 / kWords, T());
  }
};

// Two tokens of a group, A and B, and whether they count.
template <typename T>
struct Tokens {
  Raw8<T> A, B;
  bool onA, onB;

  __device__ __forceinline__ void load(const BalanceArgs& a, const T* x, long long at, int nA, int nB, int e0, int vec) {
    onA = nA < a.N && (a.mask == nullptr || a.mask[at + nA]);
    onB = nB < a.N && (a.mask == nullptr || a.mask[at + nB]);
    A.zero();
    B.zero();
    if (onA) A.load(x + nA * a.sn, e0, a.E, vec);
    if (onB) B.load(x + nB * a.sn, e0, a.E, vec);
  }
};

template <typename T>
__device__ __forceinline__ Pair<T> pair_of(float a, float b) {
  if constexpr (sizeof(T) == 2) {
    const float f[2] = {a, b};
    const uint32_t top = sizeof(T) == 2 ? (uint32_t)(ElemOf<T>::kNegInf & 0x7fffu) * 0x10001u : 0u;  // +inf
    return Pair<T>{word(__hmin2(h2(word_down(f, T()), T()), h2(top, T())))};
  } else {
    return Pair<T>{fminf(a, INFINITY), fminf(b, INFINITY)};
  }
}

template <int kLanes>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// 2^((x - m) log2 e) in place, and their sum over the token's lanes.
template <int kLanes>
__device__ __forceinline__ float exps(float (&f)[8], float m) {
  const float2 off = make_float2(-m, -m), c = make_float2(kLog2e, kLog2e);
  float2 s = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 t = __fmul2_rn(__fadd2_rn(make_float2(f[i], f[i + 1]), off), c);
    f[i] = ex2(t.x);
    f[i + 1] = ex2(t.y);
    s = __fadd2_rn(s, make_float2(f[i], f[i + 1]));
  }
  return group_sum<kLanes>(s.x + s.y);
}

// CTAs of an SM: both tokens' fp32 lists need the registers of two (three of them spill).
template <typename T, int kTop>
constexpr int kSelectCtas = sizeof(T) == 4 && kTop > 0 ? 2 : 3;

// kTop: the length of the sorted lists, at least the number of choices; 0: the choices are given.
template <typename T, int kTop, int kLog>
__global__ void __launch_bounds__(kWarps * 32, kSelectCtas<T, kTop>) balance_fwd8_kernel(BalanceArgs a, int vec) {
  __shared__ float sum_p[257];
  __shared__ int hist[257];
  const int g = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kLanes = 1 << kLog, per = 32 >> kLog;
  const int l = lane & (kLanes - 1), sub = lane >> kLog, e0 = 8 * l;
  for (int e = threadIdx.x; e <= a.E; e += blockDim.x) {
    sum_p[e] = 0.f;
    hist[e] = 0;
  }
  __syncthreads();
  float acc[8], z = 0.f;
  int count[8], tokens = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    acc[i] = 0.f;
    count[i] = 0;
  }
  const T* x = reinterpret_cast<const T*>(a.x) + g * a.sg;
  const int step = gridDim.x * kWarps * 2 * per;
  const long long at = (long long)g * a.N;
  int n0 = (blockIdx.x * kWarps + warp) * 2 * per;
  Tokens<T> ahead;
  if (n0 < a.N) ahead.load(a, x, at, n0 + sub, n0 + sub + per, e0, vec);
  for (; n0 < a.N; n0 += step) {
    const int nA = n0 + sub, nB = nA + per;
    const bool onA = ahead.onA, onB = ahead.onB;
    float fA[8], fB[8];
    ahead.A.up(fA);
    ahead.B.up(fB);
    if (n0 + step < a.N) ahead.load(a, x, at, nA + step, nB + step, e0, vec);
    const uint32_t on = (onA ? 1u : 0u) | (onB ? 0x10000u : 0u);
    float2 top;
    if constexpr (kTop > 0) {
      Pair<T> v[8], best[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) best[i] = v[i] = pair_of<T>(fA[i], fB[i]);
      sort8(best);
#pragma unroll
      for (int o = 1; o < kLanes / 2; o <<= 1) merge_top<T, kTop>(best, o);
      Pair<T> least;
      if (kLanes > 1 && a.K == kTop) {
        // Of the last merge only its ends are wanted: the smallest of the kTop largest needs no sorted list.
        Pair<T> other = from_lane(best[kTop - 1], kLanes / 2), first = best[0];
        least = larger(best[0], other);
#pragma unroll
        for (int k = 1; k < kTop; ++k) {
          other = from_lane(best[kTop - 1 - k], kLanes / 2);
          least = smaller(least, larger(best[k], other));
        }
        top = both(larger(first, other));
      } else {
        if (kLanes > 1) merge_top<T, kTop>(best, kLanes / 2);
        top = both(best[0]);
        least = best[0];
#pragma unroll
        for (int k = 1; k < kTop; ++k)
          if (k < a.K) least = best[k];
      }
      uint32_t chosen[8], total = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        chosen[i] = at_least(v[i], least) & on;
        total += chosen[i];
      }
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      if (__any_sync(0xffffffffu, total != on * (uint32_t)a.K)) {
        // More than K are at least the K-th: of those equal to it the lowest indices stay.
        uint32_t equal[8], mine = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          equal[i] = alike(v[i], least) & on;
          mine += equal[i];
        }
        uint32_t before = mine;
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) {
          const uint32_t up = __shfl_up_sync(0xffffffffu, before, o);
          if (l >= o) before += up;
        }
        const uint32_t all = __shfl_sync(0xffffffffu, before, lane | (kLanes - 1));
        before -= mine;
        // Of `all` equal ones total - K are too many; the first keep stay.
        const int keepA = (int)(all & 0xffffu) - ((int)(total & 0xffffu) - a.K);
        const int keepB = (int)(all >> 16) - ((int)(total >> 16) - a.K);
        int rankA = (int)(before & 0xffffu), rankB = (int)(before >> 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (equal[i] & 1u && rankA++ >= keepA) chosen[i] &= ~1u;
          if (equal[i] >> 16 && rankB++ >= keepB) chosen[i] &= ~0x10000u;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) count[i] += (int)((chosen[i] & 1u) + (chosen[i] >> 16));
    } else {
      float mA = fA[0], mB = fB[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) {
        mA = fmaxf(mA, fA[i]);
        mB = fmaxf(mB, fB[i]);
      }
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) {
        mA = fmaxf(mA, __shfl_xor_sync(0xffffffffu, mA, o));
        mB = fmaxf(mB, __shfl_xor_sync(0xffffffffu, mB, o));
      }
      top = make_float2(mA, mB);
      for (int k = l; k < 2 * a.K; k += kLanes) {  // the token's lanes share its choices
        const bool second = k >= a.K;
        if (second ? !onB : !onA) continue;
        const int64_t e = a.ids[(at + (second ? nB : nA)) * a.K + (second ? k - a.K : k)];
        if (e >= 0 && e < a.E)
          atomicAdd(hist + e, 1);
        else
          report_error(a.err, kErrBadArg);
      }
    }
    const float sA = exps<kLanes>(fA, top.x), sB = exps<kLanes>(fB, top.y);
    const float iA = onA ? __fdividef(1.f, sA) : 0.f, iB = onB ? __fdividef(1.f, sB) : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(fB[i], iB, fmaf(fA[i], iA, acc[i]));
    if (l == 0) {
      tokens += (onA ? 1 : 0) + (onB ? 1 : 0);
      if (a.z_coef != 0.f) {
        const float lA = fmaf(kLn2, log2f(sA), top.x), lB = fmaf(kLn2, log2f(sB), top.y);
        z += (onA ? lA * lA : 0.f) + (onB ? lB * lB : 0.f);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    for (int o = kLanes; o < 32; o <<= 1) {
      acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
      count[i] += __shfl_xor_sync(0xffffffffu, count[i], o);
    }
  z = lanes_sum(z);
  tokens = lanes_sum(tokens);
  for (int w = 0; w < kWarps; ++w) {  // in order, so that sums repeat
    if (warp == w && sub == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e0 + i < a.E) {
          sum_p[e0 + i] += acc[i];
          if (kTop > 0) hist[e0 + i] += count[i];
        }
      if (l == 0) {
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

template <typename T>
__device__ __forceinline__ void store8(T* x, int e, int E, int vec, const float (&f)[8]) {
  if (vec == 8) {
    if (e >= E) return;
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k)
      __stcs(reinterpret_cast<uint4*>(x + e) + k, raw_down<T, uint4>(f + k * kVecOf<T>));
    return;
  }
  if (vec == 4) {
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
      if (e + k >= E) continue;
      if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2*>(x + e + k) = raw_down<T, uint2>(f + k);
      else
        *reinterpret_cast<uint4*>(x + e + k) = raw_down<T, uint4>(f + k);
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (e + k < E) x[e + k] = ElemOf<T>::down(f[k]);
}

// The gradient of a token's 8 logits of this lane, in place: f are its logits, share 8 of E f_e - K.
template <int kLanes>
__device__ __forceinline__ void grad8(float (&f)[8], const float (&share)[8], float scale, float z_coef) {
  float m = f[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, f[i]);
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float s = exps<kLanes>(f, m);
  float2 d = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 8; i += 2) d = __ffma2_rn(make_float2(f[i], f[i + 1]), make_float2(share[i], share[i + 1]), d);
  const float inv = __fdividef(1.f, s);
  float shift = -group_sum<kLanes>(d.x + d.y) * inv;
  if (z_coef != 0.f) shift += 2.f * z_coef * fmaf(kLn2, log2f(s), m);
  const float2 k = make_float2(scale * inv, scale * inv), sh = make_float2(shift, shift);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 q = __fmul2_rn(__fmul2_rn(make_float2(f[i], f[i + 1]), k), __fadd2_rn(make_float2(share[i], share[i + 1]), sh));
    f[i] = q.x;
    f[i + 1] = q.y;
  }
}

template <typename T, int kLog>
__global__ void __launch_bounds__(kWarps * 32, 4) balance_bwd8_kernel(BalanceGradArgs b, int vec, int out_vec) {
  constexpr int kLanes = 1 << kLog, per = 32 >> kLog;
  const BalanceArgs& a = b.f;
  const int g = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = lane & (kLanes - 1), sub = lane >> kLog, e0 = 8 * l;
  const float* share = a.share + (long long)g * (a.E + 1);
  const float scale = b.g_loss[g * b.g_stride] * share[a.E];
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = e0 + i < a.E ? share[e0 + i] : 0.f;
  const T* x = reinterpret_cast<const T*>(a.x) + g * a.sg;
  T* out = reinterpret_cast<T*>(b.out) + (long long)g * a.N * a.E;
  const long long at = (long long)g * a.N;
  const int step = gridDim.x * kWarps * 2 * per;
  int n0 = (blockIdx.x * kWarps + warp) * 2 * per;
  Tokens<T> ahead;
  if (n0 < a.N) ahead.load(a, x, at, n0 + sub, n0 + sub + per, e0, vec);
  for (; n0 < a.N; n0 += step) {
    const int nA = n0 + sub, nB = nA + per;
    const bool onA = ahead.onA, onB = ahead.onB;
    float fA[8], fB[8];
    ahead.A.up(fA);
    ahead.B.up(fB);
    if (n0 + step < a.N) ahead.load(a, x, at, nA + step, nB + step, e0, vec);
    grad8<kLanes>(fA, f, scale, a.z_coef);
    grad8<kLanes>(fB, f, scale, a.z_coef);
    if (!onA) {  // 0, not -0 or a NaN of the scale
#pragma unroll
      for (int i = 0; i < 8; ++i) fA[i] = 0.f;
    }
    if (!onB) {
#pragma unroll
      for (int i = 0; i < 8; ++i) fB[i] = 0.f;
    }
    if (nA < a.N) store8(out + (long long)nA * a.E, e0, a.E, out_vec, fA);
    if (nB < a.N) store8(out + (long long)nB * a.E, e0, a.E, out_vec, fB);
  }
}

// ---------------------------------------------------------------- any number of experts and choices
// One token for each warp at a time; lane l holds experts l, l + 32, ...
// The simple kernels, which more than 256 experts or 8 choices reach: K rounds over the lanes, each waiting for the last
// one's maximum (ALU 74 %, 156 registers), and loads of single elements. 16 x 8192 tokens, 512 experts, top 10, bf16: forward
// 675 us where reading takes 20, backward 175 (41); 64 experts, top 16: forward 1730 us.
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

// One CTA for each group: thread (slice, expert) adds every slices-th chunk, then slices are added in order.
constexpr int kFinish = 1024;

__global__ void __launch_bounds__(kFinish) balance_finish_kernel(BalanceArgs a) {
  __shared__ double part_p[kFinish];
  __shared__ int part_n[kFinish];
  __shared__ double red[kFinish / 32];
  __shared__ double tokens;
  const int g = blockIdx.x, cells = a.E + 1;
  const long long base = (long long)g * a.chunks * cells;
  int width = 1;  // experts side by side
  while (width < cells && width < kFinish) width *= 2;
  const int slices = kFinish / width, col = threadIdx.x & (width - 1), slice = threadIdx.x / width;
  // The last cell (tokens, squares) first: its block of columns tells by how much to divide.
  double dot = 0, zz = 0, inv = 0;
  for (int e0 = (cells - 1) / width * width; e0 >= 0; e0 -= width) {
    const int e = e0 + col;
    double p = 0;
    int n = 0;
    if (e < cells) {
#pragma unroll 4
      for (int k = slice; k < a.chunks; k += slices) {
        n += a.part_count[base + (long long)k * cells + e];
        p += a.part[base + (long long)k * cells + e];
      }
    }
    part_p[threadIdx.x] = p;
    part_n[threadIdx.x] = n;
    __syncthreads();
    long long c = 0;
    if (slice == 0) {
      p = 0;
      for (int k = 0; k < slices; ++k) {
        p += part_p[k * width + col];
        c += part_n[k * width + col];
      }
      if (e == a.E) {
        tokens = (double)c;
        zz = p;
      }
    }
    __syncthreads();
    inv = 1.0 / fmax(tokens, 1.0);
    if (slice == 0 && e < a.E) {
      a.counts[(long long)g * a.E + e] = c;
      a.share[(long long)g * cells + e] = (float)(((double)a.E * c - a.K * tokens) * inv);  // whole numbers: exact before the division
      dot += c * inv * p;
    }
    if (slice == 0 && e == a.E) a.share[(long long)g * cells + a.E] = (float)inv;
  }
  // zz is with one thread only: it is added like a share of the loss.
  double v = a.E * dot * inv + (a.z_coef != 0.f ? a.z_coef * zz * inv : 0.0);
  v = lanes_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    v = 0;
    for (int k = 0; k < kFinish / 32; ++k) v += red[k];
    a.loss[g] = (float)v;
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
  for (int i = 0; i < kPer; ++i) f[i] = lane + 32 * i < a.E ? share[lane + 32 * i] : 0.f;
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

// Elements of an access to rows of E.
template <typename T>
int vec_of(const void* p, long long sg, long long sn, const BalanceArgs& a) {
  for (int vec = 8; vec >= 4; vec /= 2) {
    const int bytes = vec * (int)sizeof(T) < 16 ? vec * (int)sizeof(T) : 16;
    if (reinterpret_cast<uintptr_t>(p) % bytes == 0 && a.E % vec == 0 && (a.N <= 1 || sn * sizeof(T) % bytes == 0) &&
        (a.G <= 1 || sg * sizeof(T) % bytes == 0))
      return vec;
  }
  return 1;
}

// CTAs of a group: all groups' together stay resident (per_sm of an SM), and no warp goes without tokens.
int chunks_of(const BalanceArgs& a, int per_sm, int tokens) {
  const int want = a.G > 0 ? 148 * per_sm / a.G : 1, have = (a.N + tokens - 1) / tokens;
  return want < have ? (want < 1 ? 1 : want) : (have < 1 ? 1 : have);
}

int log_of(int E) {
  int log = 0;
  while ((8 << log) < E) ++log;
  return log;
}

// f of the lanes' exponent as a constant.
template <typename F>
void with_log(int log, F f) {
  if (log == 0) f(std::integral_constant<int, 0>());
  if (log == 1) f(std::integral_constant<int, 1>());
  if (log == 2) f(std::integral_constant<int, 2>());
  if (log == 3) f(std::integral_constant<int, 3>());
  if (log == 4) f(std::integral_constant<int, 4>());
  if (log == 5) f(std::integral_constant<int, 5>());
}

template <typename T>
void fwd_of(const BalanceArgs& a, cudaStream_t s) {
  if (a.E <= 256 && (a.ids != nullptr || a.K <= 8)) {
    const int log = log_of(a.E), vec = vec_of<T>(a.x, a.sg, a.sn, a);
    const dim3 grid(a.chunks, a.G);
    with_log(log, [&](auto k) {
      constexpr int kLog = decltype(k)::value;
      if (a.ids != nullptr)
        balance_fwd8_kernel<T, 0, kLog><<<grid, kWarps * 32, 0, s>>>(a, vec);
      else if (a.K <= 2)
        balance_fwd8_kernel<T, 2, kLog><<<grid, kWarps * 32, 0, s>>>(a, vec);
      else
        balance_fwd8_kernel<T, 8, kLog><<<grid, kWarps * 32, 0, s>>>(a, vec);
    });
    return;
  }
  if (a.E <= 256) return launch_fwd<T, 8>(a, s);
  launch_fwd<T, 32>(a, s);
}

template <typename T>
void bwd_of(const BalanceGradArgs& b, cudaStream_t s) {
  if (b.f.E <= 256) {
    const BalanceArgs& a = b.f;
    const int out_vec = vec_of<T>(b.out, (long long)a.N * a.E, a.E, a);
    const int log = log_of(a.E), tokens = kWarps * 2 * (32 >> log);
    const dim3 grid(chunks_of(a, 4, tokens), a.G);
    const int vec = vec_of<T>(a.x, a.sg, a.sn, a);
    with_log(log, [&](auto k) {
      balance_bwd8_kernel<T, decltype(k)::value><<<grid, kWarps * 32, 0, s>>>(b, vec, out_vec);
    });
    return;
  }
  launch_bwd<T, 32>(b, s);
}

}  // namespace

int balance_chunks(const BalanceArgs& a) {
  const int log = a.E <= 256 ? log_of(a.E) : 5;
  const int per_sm = a.type == Elem::kF32 && a.ids == nullptr ? kSelectCtas<float, 8> : kSelectCtas<__half, 8>;
  return chunks_of(a, per_sm, a.E <= 256 ? kWarps * 2 * (32 >> log) : kWarps);
}

void balance_fwd(const BalanceArgs& a, cudaStream_t s) {
  if (a.type == Elem::kBF16)
    fwd_of<__nv_bfloat16>(a, s);
  else if (a.type == Elem::kF16)
    fwd_of<__half>(a, s);
  else
    fwd_of<float>(a, s);
  balance_finish_kernel<<<a.G, kFinish, 0, s>>>(a);
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
