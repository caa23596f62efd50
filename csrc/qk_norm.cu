// RMS norm of each query and key head, then the rotation of its first R elements by position.
//
//     r = rsqrt(mean x^2 + eps),  n = x r,  y = n w,
//     (y_i, y_{i+R/2}) -> (y_i cos - y_{i+R/2} sin, y_{i+R/2} cos + y_i sin)     i < R / 2
// Backward, with dy the gradient rotated by the opposite angle:
//     dw = sum over tokens and heads of dy n,    dx = r (w dy - n mean(w dy n)).
// Arithmetic is fp32; the result is rounded once. r is computed again in the backward, which reads x anyway.
//
// 8 x 2048 tokens, 32 + 8 heads of 128, bf16, on one B200 (copy rate 6.55 TB/s): forward 61 us for 336 MB, backward 88 us
// for 503 MB, 5.5 and 5.7 TB/s, and 7 us for the sum of the weight gradients; all in one pass of a program 161 us. What is
// left is the latency of each step's chain (load, sum over the lanes, root, store) with the few warps that the registers
// allow (96 and 123, 27 and 22 % of the warps). The backward carries the weights' sums whether or not a weight wants them.
#include "qk_norm.cuh"

#include "tc_common.cuh"

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
  report_error(a.err, kErrBadArg);
  return p < 0 ? 0 : a.table - 1;
}

// ---------------------------------------------------------------- vectors
// VEC elements in one access of 4, 8 or 16 bytes.
template <int kBytes>
struct RawOf;
template <>
struct RawOf<16> {
  using type = uint4;
};
template <>
struct RawOf<8> {
  using type = uint2;
};
template <>
struct RawOf<4> {
  using type = uint32_t;
};

template <typename T, int VEC>
struct Chunk {
  using Raw = typename RawOf<VEC * (int)sizeof(T)>::type;
  static __device__ __forceinline__ Raw load(const T* p) { return *reinterpret_cast<const Raw*>(p); }
  static __device__ __forceinline__ void up(const Raw& r, float (&f)[VEC]) { raw_up<T>(r, f); }
  static __device__ __forceinline__ void store(T* p, const float (&f)[VEC]) {
    *reinterpret_cast<Raw*>(p) = raw_down<T, Raw>(f);
  }
};

// Which elements a lane holds: 2^log lanes share a head, lane l of them the chunks [lo, lo + VEC) and
// [hi, hi + VEC), which are rotated together while they lie in the first R elements.
template <int VEC>
struct Lanes {
  int l, sub, lo, hi;
  bool on, turns;

  __device__ Lanes(const QkNormArgs& a, int log) {
    const int lane = threadIdx.x & 31, turning = a.R / (2 * VEC);
    l = lane & ((1 << log) - 1);
    sub = lane >> log;
    on = l < a.D / (2 * VEC);
    turns = l < turning;
    lo = turns ? l * VEC : a.R + (l - turning) * 2 * VEC;
    hi = turns ? a.R / 2 + l * VEC : lo + VEC;
  }
};

template <int VEC>
__device__ __forceinline__ void load_floats(const float* p, float (&f)[VEC]) {
  constexpr int kStep = VEC >= 4 ? 4 : 2;
#pragma unroll
  for (int i = 0; i < VEC; i += kStep) {
    if constexpr (kStep == 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(p + i));
      f[i] = v.x;
      f[i + 1] = v.y;
      f[i + 2] = v.z;
      f[i + 3] = v.w;
    } else {
      const float2 v = __ldg(reinterpret_cast<const float2*>(p + i));
      f[i] = v.x;
      f[i + 1] = v.y;
    }
  }
}

template <int VEC>
__device__ __forceinline__ void load_weights(const HeadTensor& X, Elem type, const Lanes<VEC>& L, float (&w0)[VEC],
                                             float (&w1)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    w0[i] = L.on ? weight_at(X.w, type, L.lo + i) : 0.f;
    w1[i] = L.on ? weight_at(X.w, type, L.hi + i) : 0.f;
  }
}

template <int VEC>
__device__ __forceinline__ void load_angles(const QkNormArgs& a, int pos, const Lanes<VEC>& L, float (&c)[VEC],
                                            float (&s)[VEC]) {
  if (L.turns) {
    const long long at = (long long)pos * (a.R / 2) + L.lo;
    load_floats(a.cos + at, c);
    load_floats(a.sin + at, s);
    return;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    c[i] = 1.f;
    s[i] = 0.f;
  }
}

// Sums over the lanes of a head; kLog < 0: their number is known at run time only.
template <int kLog>
__device__ __forceinline__ float group_sum(float v, int log) {
  if constexpr (kLog >= 0) {
#pragma unroll
    for (int o = (1 << kLog) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  } else {
    for (int o = (1 << log) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

template <int kBytes>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  const unsigned at = (unsigned)__cvta_generic_to_shared(to);
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(kBytes) : "memory");
}

__device__ __forceinline__ float rsqrt_of(float v) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// A head of 128 takes 8 lanes with two 16-byte chunks each: half as wide chunks on 16 lanes took 1.4 times as long.
// A warp's walk over one tensor: its tasks are (token, run of per_task heads), the steps of a task
// 32 / 2^log heads each. Loading and computing walk the same steps, the loads kStages - 1 ahead.
// The next task is a fixed number of tasks away: (batch, token, part) are carried along, not divided out.
struct Walk {
  int left;  // tasks from this one on
  int b, t, part;

  __device__ Walk(unsigned first, unsigned by, unsigned tasks, int T, int parts) {
    left = first < tasks ? (int)((tasks - 1 - first) / by) + 1 : 0;
    part = (int)(first % (unsigned)parts);
    const unsigned token = first / (unsigned)parts;
    b = (int)(token / (unsigned)T);
    t = (int)(token % (unsigned)T);
  }
};

struct Stride {
  int b, t, part, T, parts;

  __device__ Stride(unsigned by, int T_, int parts_) : T(T_), parts(parts_) {
    part = (int)(by % (unsigned)parts);
    const unsigned token = by / (unsigned)parts;
    b = (int)(token / (unsigned)T);
    t = (int)(token % (unsigned)T);
  }
  __device__ __forceinline__ void next(Walk& w) const {
    --w.left;
    w.part += part;
    w.t += t;
    w.b += b;
    if (w.part >= parts) {
      w.part -= parts;
      ++w.t;
    }
    if (w.t >= T) {
      w.t -= T;
      ++w.b;
    }
  }
};

constexpr int kVecWarps = 4;
// Steps of the ring, kStages - 1 of them on their way; a lane reads back only what it copied itself, so none waits for
// another. The pass above with 2, 3 and 4 stages: 176, 159 and 170 us.
constexpr int kStages = 3;

// CTAs [0, q_blocks) walk q's tasks, the others k's.
template <typename T, int VEC, int kLog>
__global__ void __launch_bounds__(kVecWarps * 32, 5) qk_norm_fwd_vec_kernel(QkNormArgs a, int log, int per_task, int q_tasks,
                                                                            int k_tasks, int q_blocks, int k_blocks) {
  using C = Chunk<T, VEC>;
  using Raw = typename C::Raw;
  constexpr int P = VEC / 2;
  __shared__ Raw ring[kStages][2][kVecWarps * 32];
  if constexpr (kLog >= 0) log = kLog;
  const bool is_q = (int)blockIdx.x < q_blocks;
  const HeadTensor& X = is_q ? a.q : a.k;
  const unsigned block = is_q ? blockIdx.x : blockIdx.x - q_blocks, by = (is_q ? q_blocks : k_blocks) * kVecWarps;
  const int parts = max(is_q ? q_tasks : k_tasks, 1), H = X.H, step = 32 >> log;  // a tensor without heads has no tasks
  const unsigned tasks = H > 0 ? (unsigned)a.B * (unsigned)a.T * (unsigned)parts : 0;
  const Lanes<VEC> L(a, log);
  const float inv_d = 1.f / a.D, eps = a.eps;
  const Stride stride(by, max(a.T, 1), parts);
  Walk in(block * kVecWarps + (threadIdx.x >> 5), by, tasks, max(a.T, 1), parts), at = in;
  const long long x_step = X.sh * step;
  const int far = L.hi - L.lo;
  if (!L.on)  // lanes beyond the head's width read zeros
    for (int k = 0; k < kStages; ++k) ring[k][0][threadIdx.x] = ring[k][1][threadIdx.x] = Raw{};
  const T* x = nullptr;
  int in_h = 0, in_end = 0;
  auto enter = [&] {
    in_h = in.part * per_task;
    in_end = min(H, in_h + per_task);
    in_h += L.sub;
    x = reinterpret_cast<const T*>(X.in) + in.b * X.sb + in.t * X.st + in_h * X.sh + L.lo;
  };
  auto load = [&](int stage) {
    if (in.left > 0) {
      if (L.on && in_h < in_end) {
        copy_async<sizeof(Raw)>(&ring[stage][0][threadIdx.x], x);
        copy_async<sizeof(Raw)>(&ring[stage][1][threadIdx.x], x + far);
      }
      in_h += step;
      x += x_step;
      if (in_h - L.sub >= in_end) {
        stride.next(in);
        enter();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  enter();
#pragma unroll
  for (int k = 0; k < kStages - 1; ++k) load(k);
  float w0[VEC], w1[VEC];
  load_weights(X, a.wtype, L, w0, w1);
  int stage = 0;
  for (; at.left > 0; stride.next(at)) {
    float c[VEC], s[VEC];
    load_angles(a, table_row(a, at.b, at.t), L, c, s);
    // (x0 r w0) c - (x1 r w1) s = r (x0 (w0 c) - x1 (w1 s)), and the other: the products once for all heads.
    float2 w0c[P], w1s[P], w1c[P], w0s[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float2 cc = make_float2(c[2 * i], c[2 * i + 1]), sn = make_float2(s[2 * i], s[2 * i + 1]);
      const float2 u = make_float2(w0[2 * i], w0[2 * i + 1]), v = make_float2(w1[2 * i], w1[2 * i + 1]);
      w0c[i] = __fmul2_rn(u, cc);
      w1c[i] = __fmul2_rn(v, cc);
      w0s[i] = __fmul2_rn(u, sn);
      w1s[i] = __fmul2_rn(v, make_float2(-sn.x, -sn.y));
    }
    const int first = at.part * per_task, end = min(H, first + per_task);
    T* out = reinterpret_cast<T*>(X.out) + (((long long)at.b * a.T + at.t) * H + first + L.sub) * a.D + L.lo;
    for (int h = first + L.sub; h - L.sub < end; h += step, out += step * a.D) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      float f0[VEC], f1[VEC];
      C::up(ring[stage][0][threadIdx.x], f0);
      C::up(ring[stage][1][threadIdx.x], f1);
      float2 ss = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 x0 = make_float2(f0[2 * i], f0[2 * i + 1]), x1 = make_float2(f1[2 * i], f1[2 * i + 1]);
        ss = __ffma2_rn(x0, x0, ss);
        ss = __ffma2_rn(x1, x1, ss);
      }
      const float sq = group_sum<kLog>(ss.x + ss.y, log);
      load(stage == 0 ? kStages - 1 : stage - 1);  // the stage used a step ago
      const float r = rsqrt_of(fmaf(sq, inv_d, eps));
      const float2 rr = make_float2(r, r);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 x0 = make_float2(f0[2 * i], f0[2 * i + 1]), x1 = make_float2(f1[2 * i], f1[2 * i + 1]);
        const float2 y0 = __fmul2_rn(rr, __ffma2_rn(x1, w1s[i], __fmul2_rn(x0, w0c[i])));
        const float2 y1 = __fmul2_rn(rr, __ffma2_rn(x0, w0s[i], __fmul2_rn(x1, w1c[i])));
        f0[2 * i] = y0.x;
        f0[2 * i + 1] = y0.y;
        f1[2 * i] = y1.x;
        f1[2 * i + 1] = y1.y;
      }
      if (L.on && h < end) {
        C::store(out, f0);
        C::store(out + far, f1);
      }
      stage = stage == kStages - 1 ? 0 : stage + 1;
    }
  }
}

// As the forward; each CTA keeps its sums of one weight's gradient in registers and leaves them in `part`.
template <typename T, int VEC, int kLog>
__global__ void __launch_bounds__(kVecWarps * 32, 4) qk_norm_bwd_vec_kernel(QkNormGradArgs g, int log, int per_task,
                                                                            int q_tasks, int k_tasks) {
  using C = Chunk<T, VEC>;
  using Raw = typename C::Raw;
  constexpr int P = VEC / 2;
  __shared__ Raw ring[kStages][4][kVecWarps * 32];
  __shared__ float sum[kMaxHeadDim];
  if constexpr (kLog >= 0) log = kLog;
  const QkNormArgs& a = g.f;
  const bool is_q = (int)blockIdx.x < g.q_blocks;
  const HeadTensor& X = is_q ? a.q : a.k;
  const unsigned block = is_q ? blockIdx.x : blockIdx.x - g.q_blocks, by = (is_q ? g.q_blocks : g.k_blocks) * kVecWarps;
  const int parts = max(is_q ? q_tasks : k_tasks, 1), H = X.H, step = 32 >> log, warp = threadIdx.x >> 5;
  const T* grad = reinterpret_cast<const T*>(is_q ? g.gq : g.gk);
  const long long gb = is_q ? g.gqb : g.gkb, gt = is_q ? g.gqt : g.gkt, gh = is_q ? g.gqh : g.gkh;
  const unsigned tasks = H > 0 ? (unsigned)a.B * (unsigned)a.T * (unsigned)parts : 0;
  const Lanes<VEC> L(a, log);
  const float inv_d = 1.f / a.D, eps = a.eps;
  const Stride stride(by, max(a.T, 1), parts);
  Walk in(block * kVecWarps + warp, by, tasks, max(a.T, 1), parts), at = in;
  const long long x_step = X.sh * step, g_step = gh * step;
  const int far = L.hi - L.lo;
  for (int k = 0; k < kStages; ++k)  // lanes beyond the head's width, and a gradient that is not there, read zeros
    for (int u = 0; u < 4; ++u) ring[k][u][threadIdx.x] = Raw{};
  const T *x = nullptr, *gr = nullptr;
  int in_h = 0, in_end = 0;
  auto enter = [&] {
    in_h = in.part * per_task;
    in_end = min(H, in_h + per_task);
    in_h += L.sub;
    x = reinterpret_cast<const T*>(X.in) + in.b * X.sb + in.t * X.st + in_h * X.sh + L.lo;
    if (grad != nullptr) gr = grad + in.b * gb + in.t * gt + in_h * gh + L.lo;
  };
  auto load = [&](int stage) {
    if (in.left > 0) {
      if (L.on && in_h < in_end) {
        copy_async<sizeof(Raw)>(&ring[stage][0][threadIdx.x], x);
        copy_async<sizeof(Raw)>(&ring[stage][1][threadIdx.x], x + far);
        if (grad != nullptr) {
          copy_async<sizeof(Raw)>(&ring[stage][2][threadIdx.x], gr);
          copy_async<sizeof(Raw)>(&ring[stage][3][threadIdx.x], gr + far);
        }
      }
      in_h += step;
      x += x_step;
      gr += g_step;
      if (in_h - L.sub >= in_end) {
        stride.next(in);
        enter();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  enter();
#pragma unroll
  for (int k = 0; k < kStages - 1; ++k) load(k);
  float w0[VEC], w1[VEC];
  load_weights(X, a.wtype, L, w0, w1);
  float2 dw0[P], dw1[P];
#pragma unroll
  for (int i = 0; i < P; ++i) dw0[i] = dw1[i] = make_float2(0.f, 0.f);
  int stage = 0;
  for (; at.left > 0; stride.next(at)) {
    float c[VEC], s[VEC];
    load_angles(a, table_row(a, at.b, at.t), L, c, s);
    const int first = at.part * per_task, end = min(H, first + per_task);
    T* out = reinterpret_cast<T*>(X.out) + (((long long)at.b * a.T + at.t) * H + first + L.sub) * a.D + L.lo;
    for (int h = first + L.sub; h - L.sub < end; h += step, out += step * a.D) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      float f0[VEC], f1[VEC], d0[VEC], d1[VEC];
      C::up(ring[stage][0][threadIdx.x], f0);
      C::up(ring[stage][1][threadIdx.x], f1);
      Raw e0 = ring[stage][2][threadIdx.x], e1 = ring[stage][3][threadIdx.x];
      if (h >= end) e0 = e1 = Raw{};  // an older step's head: nothing for the weight's gradient
      C::up(e0, d0);
      C::up(e1, d1);
      float2 ss = make_float2(0.f, 0.f), dot = ss;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 x0 = make_float2(f0[2 * i], f0[2 * i + 1]), x1 = make_float2(f1[2 * i], f1[2 * i + 1]);
        const float2 g0 = make_float2(d0[2 * i], d0[2 * i + 1]), g1 = make_float2(d1[2 * i], d1[2 * i + 1]);
        const float2 cc = make_float2(c[2 * i], c[2 * i + 1]), sn = make_float2(s[2 * i], s[2 * i + 1]);
        const float2 z0 = __ffma2_rn(g1, sn, __fmul2_rn(g0, cc));
        const float2 z1 = __ffma2_rn(g0, make_float2(-sn.x, -sn.y), __fmul2_rn(g1, cc));
        ss = __ffma2_rn(x0, x0, ss);
        ss = __ffma2_rn(x1, x1, ss);
        dot = __ffma2_rn(__fmul2_rn(z0, make_float2(w0[2 * i], w0[2 * i + 1])), x0, dot);
        dot = __ffma2_rn(__fmul2_rn(z1, make_float2(w1[2 * i], w1[2 * i + 1])), x1, dot);
        d0[2 * i] = z0.x;
        d0[2 * i + 1] = z0.y;
        d1[2 * i] = z1.x;
        d1[2 * i + 1] = z1.y;
      }
      const float sq = group_sum<kLog>(ss.x + ss.y, log), dt = group_sum<kLog>(dot.x + dot.y, log);
      load(stage == 0 ? kStages - 1 : stage - 1);  // the stage used a step ago
      // Beyond the heads there is no norm: without eps the root of the ring's zeros would be infinite, and 0 times it a NaN
      // in the weight's gradient.
      const float r = h < end ? rsqrt_of(fmaf(sq, inv_d, eps)) : 0.f;
      const float pull = -r * r * (dt * r * inv_d);  // dx = r w dy + x pull
      const float2 rr = make_float2(r, r), pp = make_float2(pull, pull);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 x0 = make_float2(f0[2 * i], f0[2 * i + 1]), x1 = make_float2(f1[2 * i], f1[2 * i + 1]);
        const float2 z0 = __fmul2_rn(rr, make_float2(d0[2 * i], d0[2 * i + 1]));
        const float2 z1 = __fmul2_rn(rr, make_float2(d1[2 * i], d1[2 * i + 1]));
        dw0[i] = __ffma2_rn(z0, x0, dw0[i]);
        dw1[i] = __ffma2_rn(z1, x1, dw1[i]);
        const float2 y0 = __ffma2_rn(x0, pp, __fmul2_rn(z0, make_float2(w0[2 * i], w0[2 * i + 1])));
        const float2 y1 = __ffma2_rn(x1, pp, __fmul2_rn(z1, make_float2(w1[2 * i], w1[2 * i + 1])));
        f0[2 * i] = y0.x;
        f0[2 * i + 1] = y0.y;
        f1[2 * i] = y1.x;
        f1[2 * i + 1] = y1.y;
      }
      if (L.on && h < end) {
        C::store(out, f0);
        C::store(out + far, f1);
      }
      stage = stage == kStages - 1 ? 0 : stage + 1;
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    float u = i & 1 ? dw0[i / 2].y : dw0[i / 2].x, v = i & 1 ? dw1[i / 2].y : dw1[i / 2].x;
    for (int o = 16; o >= (1 << log); o >>= 1) {
      u += __shfl_xor_sync(0xffffffffu, u, o);
      v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    w0[i] = u;
    w1[i] = v;
  }
  for (int w = 0; w < kVecWarps; ++w) {  // in order, so that sums repeat
    if (warp == w && L.on && L.sub == 0) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        sum[L.lo + i] = (w ? sum[L.lo + i] : 0.f) + w0[i];
        sum[L.hi + i] = (w ? sum[L.hi + i] : 0.f) + w1[i];
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < a.D; i += blockDim.x) g.part[(long long)blockIdx.x * a.D + i] = sum[i];
}

// ---------------------------------------------------------------- any width and alignment
// One head for each warp, an element at a time: right for all, far from memory's rate. 8 x 2048 tokens, 32 + 8 heads of 30,
// bf16: forward 249 us for 79 MB (issue slots 81 %: divisions and single loads), backward 580 us for 118 MB.
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
constexpr int kSumWarps = 32;

__global__ void __launch_bounds__(kSumWarps * 32) qk_weight_sum_kernel(QkNormGradArgs g) {
  __shared__ float red[kSumWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
  const int first = blockIdx.y == 0 ? 0 : g.q_blocks, n = blockIdx.y == 0 ? g.q_blocks : g.k_blocks;
  float v = 0.f;
  if (e < g.f.D) {
#pragma unroll 4
    for (int k = warp; k < n; k += kSumWarps) v += g.part[(long long)(first + k) * g.f.D + e];
  }
  red[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && e < g.f.D) {
    v = 0.f;
#pragma unroll
    for (int k = 0; k < kSumWarps; ++k) v += red[k][lane];
    weight_put(blockIdx.y == 0 ? g.dqw : g.dkw, g.f.wtype, e, v);
  }
}

// How a call is cut into warps' tasks. vec: elements of an access, 0: the kernels that go an element at a time.
struct Plan {
  int vec, log, per_task, q_tasks, k_tasks;
};

bool fits(const QkNormArgs& a, const void* p, long long sb, long long st, long long sh, int vec, int size) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % (vec * size) == 0 && (a.B <= 1 || sb % vec == 0) &&
                          (a.T <= 1 || st % vec == 0) && sh % vec == 0);
}

Plan plan_of(const QkNormArgs& a, const QkNormGradArgs* g) {
  const int size = a.type == Elem::kF32 ? 4 : 2;
  for (int vec = 16 / size; vec >= 2; vec /= 2) {
    if (a.D % (2 * vec) || a.R % (2 * vec) || a.D / (2 * vec) > 32) continue;
    if (!fits(a, a.q.in, a.q.sb, a.q.st, a.q.sh, vec, size) || !fits(a, a.k.in, a.k.sb, a.k.st, a.k.sh, vec, size)) continue;
    if (g != nullptr && (!fits(a, g->gq, g->gqb, g->gqt, g->gqh, vec, size) ||
                         !fits(a, g->gk, g->gkb, g->gkt, g->gkh, vec, size)))
      continue;
    if ((reinterpret_cast<uintptr_t>(a.cos) | reinterpret_cast<uintptr_t>(a.sin)) % (vec >= 4 ? 16 : 8)) continue;
    Plan p{vec, 0, 0, 0, 0};
    while ((1 << p.log) < a.D / (2 * vec)) ++p.log;
    const int step = 32 >> p.log, most = a.q.H > a.k.H ? a.q.H : a.k.H;
    // Long runs of heads share their angles; short ones fill the GPU when there are few tokens.
    const long long tokens = (long long)a.B * a.T;
    p.per_task = step;
    while (p.per_task < most && tokens * ((a.q.H + a.k.H + 2 * p.per_task - 1) / (2 * p.per_task)) >= 148 * 32) p.per_task *= 2;
    p.q_tasks = (a.q.H + p.per_task - 1) / p.per_task;
    p.k_tasks = (a.k.H + p.per_task - 1) / p.per_task;
    if (tokens * (p.q_tasks > p.k_tasks ? p.q_tasks : p.k_tasks) >= (1ll << 31)) break;
    return p;
  }
  return Plan{0, 0, 1, a.q.H, a.k.H};
}

// CTAs for q and for k: as many as tasks ask for, at most `most`, shared as the heads are.
void blocks_of(const QkNormArgs& a, const Plan& p, long long most, int* q_blocks, int* k_blocks) {
  const long long tokens = (long long)a.B * a.T, per = p.vec ? kVecWarps : kWarps;
  const long long q = (tokens * p.q_tasks + per - 1) / per, k = (tokens * p.k_tasks + per - 1) / per;
  const int heads = a.q.H + a.k.H;  // neither may have any
  long long qs = most * a.q.H / (heads > 0 ? heads : 1), ks;
  qs = qs < 1 ? 1 : (qs > most - 1 ? most - 1 : qs);
  ks = most - qs;
  *q_blocks = (int)(q < qs ? (q < 1 ? 1 : q) : qs);
  *k_blocks = (int)(k < ks ? (k < 1 ? 1 : k) : ks);
}

template <typename T, int VEC, int kLog>
void fwd_vec(const QkNormArgs& a, const Plan& p, cudaStream_t s) {
  int q, k;
  blocks_of(a, p, 148 * 5, &q, &k);
  qk_norm_fwd_vec_kernel<T, VEC, kLog><<<q + k, kVecWarps * 32, 0, s>>>(a, p.log, p.per_task, p.q_tasks, p.k_tasks, q, k);
}

template <typename T, int VEC, int kLog>
void bwd_vec(const QkNormGradArgs& g, const Plan& p, cudaStream_t s) {
  qk_norm_bwd_vec_kernel<T, VEC, kLog><<<g.q_blocks + g.k_blocks, kVecWarps * 32, 0, s>>>(g, p.log, p.per_task, p.q_tasks,
                                                                                         p.k_tasks);
}

// The common head sizes (64 to 256 of whole vectors) have their sums unrolled.
#define BW_QK_DISPATCH(run, T, arg)                                            \
  constexpr int kFull = 16 / (int)sizeof(T);                                   \
  if (p.vec == kFull) {                                                        \
    if (p.log == 2) return run<T, kFull, 2>(arg, p, s);                        \
    if (p.log == 3) return run<T, kFull, 3>(arg, p, s);                        \
    if (p.log == 4) return run<T, kFull, 4>(arg, p, s);                        \
    return run<T, kFull, -1>(arg, p, s);                                       \
  }                                                                            \
  if constexpr (kFull == 8) {                                                  \
    if (p.vec == 4) return run<T, 4, -1>(arg, p, s);                           \
  }                                                                            \
  if (p.vec == 2) return run<T, 2, -1>(arg, p, s);

template <typename T>
void fwd_of(const QkNormArgs& a, cudaStream_t s) {
  const Plan p = plan_of(a, nullptr);
  BW_QK_DISPATCH(fwd_vec, T, a)
  const long long items = (long long)a.B * a.T * (a.q.H + a.k.H);
  qk_norm_fwd_kernel<T><<<(unsigned)((items + kWarps - 1) / kWarps), kWarps * 32, 0, s>>>(a);
}

template <typename T>
void bwd_of(const QkNormGradArgs& g, cudaStream_t s) {
  const Plan p = plan_of(g.f, &g);
  BW_QK_DISPATCH(bwd_vec, T, g)
  qk_norm_bwd_kernel<T><<<g.q_blocks + g.k_blocks, kWarps * 32, 0, s>>>(g);
}
#undef BW_QK_DISPATCH

}  // namespace

void qk_norm_blocks(const QkNormGradArgs& g, int* q_blocks, int* k_blocks) {
  blocks_of(g.f, plan_of(g.f, &g), 148 * 4, q_blocks, k_blocks);
}

void qk_norm_fwd(const QkNormArgs& a, cudaStream_t s) {
  if ((long long)a.B * a.T * (a.q.H + a.k.H) == 0) return;
  if (a.type == Elem::kBF16)
    fwd_of<__nv_bfloat16>(a, s);
  else if (a.type == Elem::kF16)
    fwd_of<__half>(a, s);
  else
    fwd_of<float>(a, s);
}

void qk_norm_bwd(const QkNormGradArgs& g, cudaStream_t s) {
  if (g.f.type == Elem::kBF16)
    bwd_of<__nv_bfloat16>(g, s);
  else if (g.f.type == Elem::kF16)
    bwd_of<__half>(g, s);
  else
    bwd_of<float>(g, s);
  qk_weight_sum_kernel<<<dim3((g.f.D + 31) / 32, 2), kSumWarps * 32, 0, s>>>(g);
}

}  // namespace bw
