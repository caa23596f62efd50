// Gated delta rule in chunks of 64 tokens, forward and backward.
//
// For each sequence and value head, with rows of k scaled to length one and rows of q to length `scale`:
//     S_t = exp(g_t) S_{t-1} + k_t beta_t (v_t - exp(g_t) S_{t-1}^T k_t)^T,      o_t = S_t^T q_t.
// Within a chunk let G_i be the sum of g from its start, D_ij = exp(G_i - G_j) for i >= j, L = strictly lower part of
// (K K^T) D, P = lower part of (Q K^T) D, S the state before the chunk and S' the one after it. Then
//     (I + L diag(beta)) E = V - diag(exp G) K S,     V' = diag(beta) E,
//     O = diag(exp G) Q S + P V',                     S' = exp(G_63) S + (diag(exp(G_63 - G)) K)^T V'.
// Four kernels: `prepare` (every chunk by itself: gates, lengths, P, and the inverse of the triangular matrix by forward
// substitution in fp32), `state` (chunk after chunk, columns of S split over CTAs: V' and S'), `output` (every chunk by itself).
//
// The backward goes the same way, from dO and dS':
//     dV' = P^T dO + diag(exp(G_63 - G)) K dS',       dV = (inverse)^T diag(beta) dV',
//     dS = exp(G_63) dS' + Q^T diag(exp G) dO - K^T diag(exp G) dV,                                    (`dstate`)
//     dP = lower(dO V'^T),  dL = -strictly lower(dV V'^T),
//     dQ = diag(exp G) dO S^T + (dP D) K,
//     dK = -diag(exp G) dV S^T + diag(exp(G_63 - G)) V' dS'^T + (dP D)^T Q + (dL D + (dL D)^T) K,
// and with b the logit of beta:  db_i = (1 - beta_i) dV_i . E_i.  Scaling S between two tokens scales everything that
// flows through it, so the log-decay's gradient is what leaves less what enters: with <dS', S'> for what the chunk hands on,
//     dg_t = sum_{i >= t} (q_i . dq_i - v_i . dv_i) + <dS', S'>.                                       (`inputs`)
//
// Matrix products run on 16-bit tensor instructions with fp32 sums. q, k and dO are bf16 as given, so they are exact; all
// that is computed (S, V', the inverse, P and their gradients) goes in as two bf16 halves, which keep 16 bits of 24: two products
// where one side is exact, three where both have halves (the product of the two low halves is below 2^-16 of the result).
// One half alone would round each operand by 2^-8, as much as the output's own rounding, several times over. fp16 inputs
// are two exact halves as well.
#include "delta_common.cuh"

#include <cooperative_groups.h>

namespace bw {
namespace {

namespace cg = cooperative_groups;

constexpr int kPad = 8;  // elements behind each row in shared memory: eight rows then lie in different banks
constexpr int kLdC = kChunk + kPad;

// Parts of an input element: bf16 is its own, fp16 has two.
template <typename I>
constexpr int kParts = sizeof(I) == 2 ? 1 : 2;
template <>
constexpr int kParts<__half> = 2;

// ---------------------------------------------------------------- tiles
// A matrix in shared memory: rows of `ld` elements, its low half `lo` elements behind the high one.
struct Tile {
  const bf16* p;
  int ld, lo;
};

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

template <bool kTrans>
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const bf16* p) {
  if (kTrans)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_at(p)) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_at(p)) : "memory");
}

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// acc (16 x 16 NP) += A (16 x K, from row m0) B (K x 16 NP, from column n0) of a warp. kAT: A is stored (K, M); kBT: B is
// stored (N, K). kA and kB: parts of each.
template <int NP, int K, bool kAT, bool kBT, int kA, int kB>
__device__ __forceinline__ void product(float (&acc)[2 * NP][4], const Tile& A, int m0, const Tile& B, int n0) {
  const int lane = threadIdx.x & 31;
  const bf16* a = kAT ? A.p + ((lane >> 4) * 8 + (lane & 7)) * A.ld + m0 + ((lane >> 3) & 1) * 8
                      : A.p + (m0 + (lane & 15)) * A.ld + (lane >> 4) * 8;
  const bf16* b = kBT ? B.p + (n0 + (lane >> 4) * 8 + (lane & 7)) * B.ld + ((lane >> 3) & 1) * 8
                      : B.p + (((lane >> 3) & 1) * 8 + (lane & 7)) * B.ld + n0 + (lane >> 4) * 8;
  const int step_a = kAT ? 16 * A.ld : 16, step_b = kBT ? 16 : 16 * B.ld;
#pragma unroll
  for (int k = 0; k < K / 16; ++k) {
    uint32_t ah[4], al[4];
    ldmatrix4<kAT>(ah, a + k * step_a);
    if (kA == 2) ldmatrix4<kAT>(al, a + A.lo + k * step_a);
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const bf16* bn = b + k * step_b + (kBT ? n * 16 * B.ld : n * 16);
      uint32_t bh[4], bl[4];
      ldmatrix4<!kBT>(bh, bn);
      if (kB == 2) ldmatrix4<!kBT>(bl, bn + B.lo);
      mma(acc[2 * n], ah, bh[0], bh[1]);
      mma(acc[2 * n + 1], ah, bh[2], bh[3]);
      if (kB == 2) {
        mma(acc[2 * n], ah, bl[0], bl[1]);
        mma(acc[2 * n + 1], ah, bl[2], bl[3]);
      }
      if (kA == 2) {
        mma(acc[2 * n], al, bh[0], bh[1]);
        mma(acc[2 * n + 1], al, bh[2], bh[3]);
      }
    }
  }
}

// Two neighbouring values as words of their high and low halves.
__device__ __forceinline__ void halves(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  const float2 f = __bfloat1622float2(h);
  const __nv_bfloat162 l = __floats2bfloat162_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

__device__ __forceinline__ void put2(bf16* p, int lo, float x, float y) {
  uint32_t h, l;
  halves(x, y, h, l);
  *reinterpret_cast<uint32_t*>(p) = h;
  *reinterpret_cast<uint32_t*>(p + lo) = l;
}

__device__ __forceinline__ float2 get2(const bf16* p, int lo) {
  const float2 h = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p));
  const float2 l = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p + lo));
  return make_float2(h.x + l.x, h.y + l.y);
}

// ---------------------------------------------------------------- loads
__device__ __forceinline__ void copy16(bf16* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_at(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory"); }

// rows x width of two planes in global memory (rows of `ldg`, the low plane `log` elements behind) into shared memory.
// Columns from `width` to kCols are zero.
template <int kCols>
__device__ __forceinline__ void load_planes(bf16* to, int ld, int lo, const bf16* from, int rows, int width, int ldg, long long log) {
  constexpr int kV = kCols / 8;
  for (int i = threadIdx.x; i < 2 * rows * kV; i += blockDim.x) {
    const int half = i / (rows * kV), r = i / kV % rows, c = i % kV * 8;
    bf16* t = to + half * lo + r * ld + c;
    if (c < width) copy16(t, from + half * log + (long long)r * ldg + c);
    else *reinterpret_cast<uint4*>(t) = make_uint4(0, 0, 0, 0);
  }
}

// Rows [0, rows) of a chunk of head rows (64 x width) into shared memory, zeros behind them and from `width` on.
template <typename I, int kCols>
__device__ __forceinline__ void load_rows(bf16* to, int ld, int lo, const I* from, long long st, int rows, int width, bool wide) {
  constexpr int kV = kCols / 8;
  for (int i = threadIdx.x; i < kChunk * kV; i += blockDim.x) {
    const int r = i / kV, c = i % kV * 8;
    bf16* t = to + r * ld + c;
    if (r >= rows || c >= width) {
      *reinterpret_cast<uint4*>(t) = make_uint4(0, 0, 0, 0);
      if (kParts<I> == 2) *reinterpret_cast<uint4*>(t + lo) = make_uint4(0, 0, 0, 0);
      continue;
    }
    const I* x = from + r * st + c;
    if constexpr (kParts<I> == 1) {
      if (wide) {
        copy16(t, x);
        continue;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) t[k] = x[k];
    } else {
      float f[8];
      if (wide) {
        raw_up<I>(__ldg(reinterpret_cast<const uint4*>(x)), f);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = ElemOf<I>::up(x[k]);
      }
#pragma unroll
      for (int k = 0; k < 8; k += 2) put2(t + k, lo, f[k], f[k + 1]);
    }
  }
}

template <typename I>
__device__ __forceinline__ float2 pair_of(const I* p, bool wide) {
  if (!wide) return make_float2(ElemOf<I>::up(p[0]), ElemOf<I>::up(p[1]));
  float f[2];
  word_up(*reinterpret_cast<const uint32_t*>(p), f, I());
  return make_float2(f[0], f[1]);
}

template <typename I>
__device__ __forceinline__ const I* head_at(const HeadRows& x, int b, long long t, int h) {
  return reinterpret_cast<const I*>(x.p) + b * x.sb + t * x.st + h * x.sh;
}

// exp(G_i - G_j) of sums held in two parts: the small part counts where the large ones nearly cancel.
__device__ __forceinline__ float decay_between(float2 i, float2 j) { return expf((i.x - j.x) + (i.y - j.y)); }

struct Place3 {
  int b, h, c;
  long long bh, n;
  __device__ Place3(const DeltaDims& d, long long head, int chunk) : c(chunk), bh(head), n(head * d.chunks + chunk) {
    b = (int)(head / d.H);
    h = (int)(head % d.H);
  }
};

// ---------------------------------------------------------------- prepare
// One chunk of one value head: 4 warps, 16 tokens' rows of both products each.
template <typename I, int DK>
__global__ void __launch_bounds__(128) prepare_kernel(const DeltaFwd a) {
  constexpr int ld = DK + kPad, plane = kChunk * ld, ldA = kChunk + 4;
  extern __shared__ __align__(16) unsigned char raw[];
  bf16* Q = reinterpret_cast<bf16*>(raw);
  bf16* K = Q + kParts<I> * plane;
  float* A = reinterpret_cast<float*>(K + kParts<I> * plane);  // (64, ldA): L diag(beta)
  __shared__ float2 G[kChunk];
  __shared__ float beta[kChunk], rk[kChunk], rq[kChunk], logs[kChunk];
  const DeltaDims& d = a.d;
  const Place3 at(d, blockIdx.x / d.chunks, blockIdx.x % d.chunks);
  const int group = d.H / d.Hk, hk = at.h / group;
  const int t0 = at.c * kChunk, rows = min(kChunk, d.T - t0);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  load_rows<I, DK>(Q, ld, plane, head_at<I>(a.q, at.b, t0, hk), a.q.st, rows, d.dk, d.wide);
  load_rows<I, DK>(K, ld, plane, head_at<I>(a.k, at.b, t0, hk), a.k.st, rows, d.dk, d.wide);
  if (tid < kChunk) {
    float g = 0.f, w = 0.f;
    if (tid < rows) {
      g = gate_of(ElemOf<I>::up(*head_at<I>(a.g.a, at.b, t0 + tid, at.h)), load_any(a.g.a_log, a.g.a_log_type, at.h),
                  load_any(a.g.dt_bias, a.g.dt_bias_type, at.h)).log_decay;
      w = sigmoid(ElemOf<I>::up(*head_at<I>(a.g.b, at.b, t0 + tid, at.h)));
    }
    logs[tid] = g;
    beta[tid] = w;
    a.keep.beta[at.n * kChunk + tid] = w;
  }
  copies_done();
  __syncthreads();
  if (warp == 0) {  // sums of log-decays in 64 bits, kept as two floats
    const double x = logs[2 * lane], y = logs[2 * lane + 1];
    double sum = x + y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const double v = k ? sum : sum - y;
      const float hi = (float)v;
      const float2 g = make_float2(hi, (float)(v - hi));
      G[2 * lane + k] = g;
      a.keep.total[at.n * kChunk + 2 * lane + k] = g;
    }
  }
  for (int r = warp; r < 2 * kChunk; r += 4) {  // lengths
    const bf16* x = (r < kChunk ? K : Q) + (r % kChunk) * ld;
    float sq = 0.f;
    for (int i = lane * 2; i < DK; i += 64) {
      float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(x + i));
      if (kParts<I> == 2) v = get2(x + i, plane);
      sq = fmaf(v.x, v.x, fmaf(v.y, v.y, sq));
    }
    sq = lanes_sum(sq);
    const float len = rsqrtf(sq + 1e-6f);
    if (lane == 0) (r < kChunk ? rk[r] : rq[r - kChunk]) = r < kChunk ? len : len * d.scale;
  }
  float kk[8][4], qk[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) kk[i][j] = qk[i][j] = 0.f;
  const Tile tk{K, ld, plane}, tq{Q, ld, plane};
  product<4, DK, false, true, kParts<I>, kParts<I>>(kk, tk, warp * 16, tk, 0);
  product<4, DK, false, true, kParts<I>, kParts<I>>(qk, tq, warp * 16, tk, 0);
  __syncthreads();
  bf16* P = a.keep.attend + at.n * 2 * kChunk * kChunk;
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const int i = warp * 16 + (lane >> 2) + (e ? 8 : 0), j = n * 8 + (lane & 3) * 2;
      float p[2], l[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float w = j + x <= i ? decay_between(G[i], G[j + x]) * rk[j + x] : 0.f;
        p[x] = j + x <= i ? qk[n][e + x] * rq[i] * w : 0.f;
        l[x] = j + x < i ? kk[n][e + x] * rk[i] * w * beta[j + x] : 0.f;
      }
      put2(P + i * kChunk + j, kChunk * kChunk, p[0], p[1]);
      *reinterpret_cast<float2*>(A + i * ldA + j) = make_float2(l[0], l[1]);
    }
  __syncthreads();
  if (tid < kChunk) {
    const long long m = ((long long)at.b * d.Hk + hk) * d.chunks + at.c;
    if (at.h % group == 0) {
      a.keep.rk[m * kChunk + tid] = rk[tid];
      a.keep.rq[m * kChunk + tid] = rq[tid];
    }
    // Column `tid` of the inverse: x_i = [i = tid] - sum_{m < i} A_im x_m.
    bf16* X = a.keep.solve + at.n * 2 * kChunk * kChunk + tid;
    float x[kChunk];
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      float s[4] = {i == tid ? 1.f : 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int m = 0; m < i; ++m) s[m & 3] = fmaf(-A[i * ldA + m], x[m], s[m & 3]);
      x[i] = (s[0] + s[1]) + (s[2] + s[3]);
      const bf16 h = __float2bfloat16_rn(x[i]);
      X[i * kChunk] = h;
      X[kChunk * kChunk + i * kChunk] = __float2bfloat16_rn(x[i] - __bfloat162float(h));
    }
  }
}

// ---------------------------------------------------------------- state
// NV columns of a head's state, chunk after chunk. 8 warps: 4 x 2 over (tokens, columns), DK / 16 x the rest over (rows, columns).
template <typename I, int DK, int NV>
__global__ void __launch_bounds__(256) state_kernel(const DeltaFwd a) {
  constexpr int ldk = DK + kPad, planeK = kChunk * ldk, ldv = NV + kPad, planeS = DK * ldv, planeX = kChunk * ldv,
                planeC = kChunk * kLdC;
  constexpr int kMW = DK / 16, kNW = 8 / kMW, kNP = NV / 32, kSP = NV / 16 / kNW;
  extern __shared__ __align__(16) unsigned char raw[];
  bf16* K = reinterpret_cast<bf16*>(raw);
  bf16* X = K + kParts<I> * planeK;   // the right-hand side, then the scaled writes
  bf16* S = X + 2 * planeX;
  bf16* C = S + 2 * planeS;           // the inverse
  const DeltaDims& d = a.d;
  const int slices = (d.dv + NV - 1) / NV, v0 = blockIdx.x % slices * NV, width = min(NV, d.dv - v0);
  const long long head = blockIdx.x / slices;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t2 = (lane & 3) * 2;
  const int m0 = warp % 4 * 16, n0 = warp / 4 * (NV / 2);       // of (tokens, columns)
  const int sm0 = warp % kMW * 16, sn0 = warp / kMW * (NV / kNW);  // of (rows, columns) of the state
  float st[2 * kSP][4];
#pragma unroll
  for (int n = 0; n < 2 * kSP; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = sm0 + g + (e / 2) * 8, c = sn0 + n * 8 + t2 + (e & 1);
      st[n][e] = a.first != nullptr && r < d.dk && c < width ? a.first[(head * d.dk + r) * d.dv + v0 + c] : 0.f;
    }
  const Tile tK{K, ldk, planeK}, tX{X, ldv, planeX}, tS{S, ldv, planeS}, tC{C, kLdC, planeC};
  for (int c = 0; c <= d.chunks; ++c) {
    const Place3 at(d, head, c);
    // The state before the chunk, for this kernel's products and for the others'.
    bf16* keep = a.keep.states + (head * (d.chunks + 1) + c) * 2 * d.dk * d.dv;
#pragma unroll
    for (int n = 0; n < 2 * kSP; ++n)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const int r = sm0 + g + e * 4, col = sn0 + n * 8 + t2;
        uint32_t h, l;
        halves(st[n][e], st[n][e + 1], h, l);
        *reinterpret_cast<uint32_t*>(S + r * ldv + col) = h;
        *reinterpret_cast<uint32_t*>(S + planeS + r * ldv + col) = l;
        if (r < d.dk && col < width) {
          *reinterpret_cast<uint32_t*>(keep + r * d.dv + v0 + col) = h;
          *reinterpret_cast<uint32_t*>(keep + (long long)d.dk * d.dv + r * d.dv + v0 + col) = l;
        }
      }
    if (c == d.chunks) break;
    const int hk = at.h / (d.H / d.Hk), t0 = c * kChunk, rows = min(kChunk, d.T - t0);
    load_rows<I, DK>(K, ldk, planeK, head_at<I>(a.k, at.b, t0, hk), a.k.st, rows, d.dk, d.wide);
    load_planes<kChunk>(C, kLdC, planeC, a.keep.solve + at.n * 2 * kChunk * kChunk, kChunk, kChunk, kChunk, kChunk * kChunk);
    const long long m = ((long long)at.b * d.Hk + hk) * d.chunks + c;
    const float2 end = a.keep.total[at.n * kChunk + kChunk - 1];
    float in[2], beta[2], out[2];  // of the thread's two tokens: exp(G) rk, beta, exp(G_63 - G) rk
    float2 v[2 * kNP][2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = m0 + g + k * 8;
      const float2 G = a.keep.total[at.n * kChunk + i];
      const float rk = a.keep.rk[m * kChunk + i];
      in[k] = expf(G.x + G.y) * rk;
      out[k] = decay_between(end, G) * rk;
      beta[k] = a.keep.beta[at.n * kChunk + i];
#pragma unroll
      for (int n = 0; n < 2 * kNP; ++n) {
        const int col = n0 + n * 8 + t2;
        v[n][k] = i < rows && col < width ? pair_of(head_at<I>(a.v, at.b, t0 + i, at.h) + v0 + col, d.wide) : make_float2(0.f, 0.f);
      }
    }
    copies_done();
    __syncthreads();
    float acc[2 * kNP][4];
#pragma unroll
    for (int n = 0; n < 2 * kNP; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
    product<kNP, DK, false, false, kParts<I>, 2>(acc, tK, m0, tS, n0);
#pragma unroll
    for (int n = 0; n < 2 * kNP; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        put2(X + (m0 + g + k * 8) * ldv + n0 + n * 8 + t2, planeX, fmaf(-in[k], acc[n][2 * k], v[n][k].x),
             fmaf(-in[k], acc[n][2 * k + 1], v[n][k].y));
        acc[n][2 * k] = acc[n][2 * k + 1] = 0.f;
      }
    __syncthreads();
    product<kNP, kChunk, false, false, 2, 2>(acc, tC, m0, tX, n0);
    __syncthreads();
    bf16* writes = a.keep.writes + at.n * 2 * kChunk * d.dv + v0;
#pragma unroll
    for (int n = 0; n < 2 * kNP; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int i = m0 + g + k * 8, col = n0 + n * 8 + t2;
        const float x = acc[n][2 * k] * beta[k], y = acc[n][2 * k + 1] * beta[k];
        if (col < width) put2(writes + i * d.dv + col, kChunk * d.dv, x, y);
        put2(X + i * ldv + col, planeX, x * out[k], y * out[k]);
      }
    const float left = expf(end.x + end.y);
#pragma unroll
    for (int n = 0; n < 2 * kSP; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) st[n][e] *= left;
    __syncthreads();
    product<kSP, kChunk, true, false, kParts<I>, 2>(st, tK, sm0, tX, sn0);
    __syncthreads();
  }
  if (a.last != nullptr) {
#pragma unroll
    for (int n = 0; n < 2 * kSP; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = sm0 + g + (e / 2) * 8, c = sn0 + n * 8 + t2 + (e & 1);
        if (r < d.dk && c < width) a.last[(head * d.dk + r) * d.dv + v0 + c] = st[n][e];
      }
  }
}

// ---------------------------------------------------------------- output
// NV columns of a chunk's output. 8 warps: 4 x 2 over (tokens, columns).
template <typename I, int DK, int NV>
__global__ void __launch_bounds__(256) output_kernel(const DeltaFwd a) {
  constexpr int ldk = DK + kPad, planeK = kChunk * ldk, ldv = NV + kPad, planeS = DK * ldv, planeX = kChunk * ldv,
                planeC = kChunk * kLdC, kNP = NV / 32;
  extern __shared__ __align__(16) unsigned char raw[];
  bf16* Q = reinterpret_cast<bf16*>(raw);
  bf16* X = Q + kParts<I> * planeK;
  bf16* S = X + 2 * planeX;
  bf16* C = S + 2 * planeS;
  const DeltaDims& d = a.d;
  const int slices = (d.dv + NV - 1) / NV, v0 = blockIdx.x % slices * NV, width = min(NV, d.dv - v0);
  const long long n_ = blockIdx.x / slices;
  const Place3 at(d, n_ / d.chunks, (int)(n_ % d.chunks));
  const int hk = at.h / (d.H / d.Hk), t0 = at.c * kChunk, rows = min(kChunk, d.T - t0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t2 = (lane & 3) * 2;
  const int m0 = warp % 4 * 16, n0 = warp / 4 * (NV / 2);
  load_rows<I, DK>(Q, ldk, planeK, head_at<I>(a.q, at.b, t0, hk), a.q.st, rows, d.dk, d.wide);
  load_planes<kChunk>(C, kLdC, planeC, a.keep.attend + at.n * 2 * kChunk * kChunk, kChunk, kChunk, kChunk, kChunk * kChunk);
  load_planes<NV>(X, ldv, planeX, a.keep.writes + at.n * 2 * kChunk * d.dv + v0, kChunk, width, d.dv, (long long)kChunk * d.dv);
  load_planes<NV>(S, ldv, planeS, a.keep.states + (at.bh * (d.chunks + 1) + at.c) * 2 * d.dk * d.dv + v0, d.dk, width, d.dv,
                  (long long)d.dk * d.dv);
  for (int i = threadIdx.x; i < 2 * (DK - d.dk) * ldv; i += blockDim.x)  // rows behind the head's width
    S[i / ((DK - d.dk) * ldv) * planeS + d.dk * ldv + i % ((DK - d.dk) * ldv)] = __float2bfloat16_rn(0.f);
  const long long m = ((long long)at.b * d.Hk + hk) * d.chunks + at.c;
  float in[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = m0 + g + k * 8;
    const float2 G = a.keep.total[at.n * kChunk + i];
    in[k] = expf(G.x + G.y) * a.keep.rq[m * kChunk + i];
  }
  copies_done();
  __syncthreads();
  float acc[2 * kNP][4];
#pragma unroll
  for (int n = 0; n < 2 * kNP; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
  const Tile tQ{Q, ldk, planeK}, tX{X, ldv, planeX}, tS{S, ldv, planeS}, tC{C, kLdC, planeC};
  product<kNP, DK, false, false, kParts<I>, 2>(acc, tQ, m0, tS, n0);
#pragma unroll
  for (int n = 0; n < 2 * kNP; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[n][e] *= in[e / 2];
  product<kNP, kChunk, false, false, 2, 2>(acc, tC, m0, tX, n0);
  I* out = reinterpret_cast<I*>(a.out);
#pragma unroll
  for (int n = 0; n < 2 * kNP; ++n)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = m0 + g + k * 8, col = n0 + n * 8 + t2;
      if (i < rows && col < width)
        *reinterpret_cast<uint32_t*>(out + (((long long)at.b * d.T + t0 + i) * d.H + at.h) * d.dv + v0 + col) =
            word_down(&acc[n][2 * k], I());
    }
}

// ---------------------------------------------------------------- dstate
// NV columns of the gradient of a head's state, from the last chunk to the first.
template <typename I, int DK, int NV>
__global__ void __launch_bounds__(256) dstate_kernel(const DeltaBwd a) {
  constexpr int ldk = DK + kPad, planeK = kChunk * ldk, ldv = NV + kPad, planeS = DK * ldv, planeX = kChunk * ldv,
                planeC = kChunk * kLdC;
  constexpr int kMW = DK / 16, kNW = 8 / kMW, kNP = NV / 32, kSP = NV / 16 / kNW;
  extern __shared__ __align__(16) unsigned char raw[];
  bf16* K = reinterpret_cast<bf16*>(raw);
  bf16* Q = K + kParts<I> * planeK;
  bf16* O = Q + kParts<I> * planeK;   // dO
  bf16* Y = O + kParts<I> * planeX;   // diag(exp G rq) dO
  bf16* X = Y + 2 * planeX;           // beta dV', then -diag(exp G rk) dV
  bf16* S = X + 2 * planeX;
  bf16* C = S + 2 * planeS;           // P
  bf16* R = C + 2 * planeC;           // the inverse
  const DeltaDims& d = a.d;
  const int slices = (d.dv + NV - 1) / NV, v0 = blockIdx.x % slices * NV, width = min(NV, d.dv - v0);
  const long long head = blockIdx.x / slices;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t2 = (lane & 3) * 2;
  const int m0 = warp % 4 * 16, n0 = warp / 4 * (NV / 2);
  const int sm0 = warp % kMW * 16, sn0 = warp / kMW * (NV / kNW);
  float st[2 * kSP][4];
#pragma unroll
  for (int n = 0; n < 2 * kSP; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = sm0 + g + (e / 2) * 8, c = sn0 + n * 8 + t2 + (e & 1);
      st[n][e] = a.g_last != nullptr && r < d.dk && c < width ? a.g_last[(head * d.dk + r) * d.dv + v0 + c] : 0.f;
    }
  const Tile tK{K, ldk, planeK}, tQ{Q, ldk, planeK}, tO{O, ldv, planeX}, tY{Y, ldv, planeX}, tX{X, ldv, planeX},
      tS{S, ldv, planeS}, tC{C, kLdC, planeC}, tR{R, kLdC, planeC};
  const I* g_out = reinterpret_cast<const I*>(a.g_out);
  I* dv = reinterpret_cast<I*>(a.dv);
  for (int c = d.chunks - 1; c >= 0; --c) {
    const Place3 at(d, head, c);
    bf16* keep = a.dstates + at.n * 2 * d.dk * d.dv;
#pragma unroll
    for (int n = 0; n < 2 * kSP; ++n)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const int r = sm0 + g + e * 4, col = sn0 + n * 8 + t2;
        uint32_t h, l;
        halves(st[n][e], st[n][e + 1], h, l);
        *reinterpret_cast<uint32_t*>(S + r * ldv + col) = h;
        *reinterpret_cast<uint32_t*>(S + planeS + r * ldv + col) = l;
        if (r < d.dk && col < width) {
          *reinterpret_cast<uint32_t*>(keep + r * d.dv + v0 + col) = h;
          *reinterpret_cast<uint32_t*>(keep + (long long)d.dk * d.dv + r * d.dv + v0 + col) = l;
        }
      }
    const int hk = at.h / (d.H / d.Hk), t0 = c * kChunk, rows = min(kChunk, d.T - t0);
    const long long m = ((long long)at.b * d.Hk + hk) * d.chunks + c;
    load_rows<I, DK>(K, ldk, planeK, head_at<I>(a.k, at.b, t0, hk), a.k.st, rows, d.dk, d.wide);
    load_rows<I, DK>(Q, ldk, planeK, head_at<I>(a.q, at.b, t0, hk), a.q.st, rows, d.dk, d.wide);
    const I* go = g_out + (((long long)at.b * d.T + t0) * d.H + at.h) * d.dv + v0;
    load_rows<I, NV>(O, ldv, planeX, go, (long long)d.H * d.dv, rows, width, true);
    load_planes<kChunk>(C, kLdC, planeC, a.keep.attend + at.n * 2 * kChunk * kChunk, kChunk, kChunk, kChunk, kChunk * kChunk);
    load_planes<kChunk>(R, kLdC, planeC, a.keep.solve + at.n * 2 * kChunk * kChunk, kChunk, kChunk, kChunk, kChunk * kChunk);
    const float2 end = a.keep.total[at.n * kChunk + kChunk - 1];
    float in[2], beta[2], out[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = m0 + g + k * 8;
      const float2 G = a.keep.total[at.n * kChunk + i];
      const float rk = a.keep.rk[m * kChunk + i], grown = expf(G.x + G.y), fq = grown * a.keep.rq[m * kChunk + i];
      in[k] = grown * rk;
      out[k] = decay_between(end, G) * rk;
      beta[k] = a.keep.beta[at.n * kChunk + i];
#pragma unroll
      for (int n = 0; n < 2 * kNP; ++n) {
        const int col = n0 + n * 8 + t2;
        const float2 x = i < rows && col < width ? pair_of(go + (long long)i * d.H * d.dv + col, true) : make_float2(0.f, 0.f);
        put2(Y + i * ldv + col, planeX, x.x * fq, x.y * fq);
      }
    }
    copies_done();
    __syncthreads();
    float acc[2 * kNP][4];
#pragma unroll
    for (int n = 0; n < 2 * kNP; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
    product<kNP, DK, false, false, kParts<I>, 2>(acc, tK, m0, tS, n0);
#pragma unroll
    for (int n = 0; n < 2 * kNP; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] *= out[e / 2];
    product<kNP, kChunk, true, false, 2, kParts<I>>(acc, tC, m0, tO, n0);
#pragma unroll
    for (int n = 0; n < 2 * kNP; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        put2(X + (m0 + g + k * 8) * ldv + n0 + n * 8 + t2, planeX, acc[n][2 * k] * beta[k], acc[n][2 * k + 1] * beta[k]);
        acc[n][2 * k] = acc[n][2 * k + 1] = 0.f;
      }
    __syncthreads();
    product<kNP, kChunk, true, false, 2, 2>(acc, tR, m0, tX, n0);
    __syncthreads();
    bf16* reads = a.dreads + at.n * 2 * kChunk * d.dv + v0;
#pragma unroll
    for (int n = 0; n < 2 * kNP; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int i = m0 + g + k * 8, col = n0 + n * 8 + t2;
        if (col < width) {
          put2(reads + i * d.dv + col, kChunk * d.dv, acc[n][2 * k], acc[n][2 * k + 1]);
          if (i < rows)
            *reinterpret_cast<uint32_t*>(dv + (((long long)at.b * d.T + t0 + i) * d.H + at.h) * d.dv + v0 + col) =
                word_down(&acc[n][2 * k], I());
        }
        put2(X + i * ldv + col, planeX, -acc[n][2 * k] * in[k], -acc[n][2 * k + 1] * in[k]);
      }
    const float left = expf(end.x + end.y);
#pragma unroll
    for (int n = 0; n < 2 * kSP; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) st[n][e] *= left;
    __syncthreads();
    product<kSP, kChunk, true, false, kParts<I>, 2>(st, tK, sm0, tX, sn0);
    product<kSP, kChunk, true, false, kParts<I>, 2>(st, tQ, sm0, tY, sn0);
    __syncthreads();
  }
  if (a.dfirst != nullptr) {
#pragma unroll
    for (int n = 0; n < 2 * kSP; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = sm0 + g + (e / 2) * 8, c = sn0 + n * 8 + t2 + (e & 1);
        if (r < d.dk && c < width) a.dfirst[(head * d.dk + r) * d.dv + v0 + c] = st[n][e];
      }
  }
}

// ---------------------------------------------------------------- inputs
// The gradients of q, k and the gates of one chunk: a CTA for each value head, the heads of one key head a cluster, whose
// CTAs add their rows of dq and dk over distributed shared memory in the order of the heads.
template <typename I, int DK>
__global__ void __launch_bounds__(256) inputs_kernel(const DeltaBwd a) {
  constexpr int NV = 32, ldk = DK + kPad, planeK = kChunk * ldk, ldv = NV + kPad, planeS = DK * ldv, planeX = kChunk * ldv,
                planeC = kChunk * kLdC, kNP = DK / 32, ldF = DK + 4;
  extern __shared__ __align__(16) unsigned char raw[];
  bf16* Q = reinterpret_cast<bf16*>(raw);
  bf16* K = Q + kParts<I> * planeK;
  bf16* O = K + kParts<I> * planeK;  // slices of dO, V', dV and a state
  bf16* W = O + kParts<I> * planeX;
  bf16* R = W + 2 * planeX;
  bf16* S = R + 2 * planeX;
  bf16* C = O;                       // then (64, 64): dP D, and the symmetric dL D
  bf16* N = C + 2 * planeC;
  float* F = reinterpret_cast<float*>(raw);  // then the cluster's exchange: dq and dk of this head (2, 64, ldF)
  __shared__ float2 G[kChunk];
  __shared__ float rk[kChunk], rq[kChunk], dots[3][kChunk], state_dot[8];
  const DeltaDims& d = a.d;
  const int group = d.H / d.Hk;
  // blockIdx.x = (batch * Hk + key head, chunk, head within the group): the last runs over the cluster
  const int hg = blockIdx.x % group;
  const long long rest = blockIdx.x / group;
  const int c = (int)(rest % d.chunks);
  const long long bk = rest / d.chunks;
  const int b = (int)(bk / d.Hk), hk = (int)(bk % d.Hk), h = hk * group + hg;
  const Place3 at(d, (long long)b * d.H + h, c);
  const int t0 = c * kChunk, rows = min(kChunk, d.T - t0);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t2 = (lane & 3) * 2;
  const int m0 = warp % 4 * 16, n0 = warp / 4 * (DK / 2), p0 = warp / 4 * 32;
  load_rows<I, DK>(Q, ldk, planeK, head_at<I>(a.q, b, t0, hk), a.q.st, rows, d.dk, d.wide);
  load_rows<I, DK>(K, ldk, planeK, head_at<I>(a.k, b, t0, hk), a.k.st, rows, d.dk, d.wide);
  const long long m = bk * d.chunks + c;
  if (tid < kChunk) {
    G[tid] = a.keep.total[at.n * kChunk + tid];
    rk[tid] = a.keep.rk[m * kChunk + tid];
    rq[tid] = a.keep.rq[m * kChunk + tid];
    dots[0][tid] = dots[1][tid] = dots[2][tid] = 0.f;
  }
  float dq[2 * kNP][4], dk[2 * kNP][4], dp[4][4], dl[4][4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
#pragma unroll
    for (int n = 0; n < 2 * kNP; ++n) dq[n][e] = dk[n][e] = 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n) dp[n][e] = dl[n][e] = 0.f;
  }
  const Tile tK{K, ldk, planeK}, tQ{Q, ldk, planeK}, tO{O, ldv, planeX}, tW{W, ldv, planeX}, tR{R, ldv, planeX}, tS{S, ldv, planeS},
      tC{C, kLdC, planeC}, tN{N, kLdC, planeC};
  const I* g_out = reinterpret_cast<const I*>(a.g_out) + (((long long)b * d.T + t0) * d.H + h) * d.dv;
  const bf16* states = a.keep.states + (at.bh * (d.chunks + 1) + c) * 2 * d.dk * d.dv;
  const bf16 *writes = a.keep.writes + at.n * 2 * kChunk * d.dv, *reads = a.dreads + at.n * 2 * kChunk * d.dv;
  const long long planeG = (long long)d.dk * d.dv;
  if (d.dk < DK)  // rows behind the head's width
    for (int i = tid; i < 2 * (DK - d.dk) * ldv; i += blockDim.x)
      S[i / ((DK - d.dk) * ldv) * planeS + d.dk * ldv + i % ((DK - d.dk) * ldv)] = __float2bfloat16_rn(0.f);
  // 1. What meets the state before the chunk: dP, dL, dQ, and dK through dV; the sums over columns of the gates' gradients.
  for (int v0 = 0; v0 < d.dv; v0 += NV) {
    const int width = min(NV, d.dv - v0);
    __syncthreads();
    load_rows<I, NV>(O, ldv, planeX, g_out + v0, (long long)d.H * d.dv, rows, width, true);
    load_planes<NV>(W, ldv, planeX, writes + v0, kChunk, width, d.dv, (long long)kChunk * d.dv);
    load_planes<NV>(R, ldv, planeX, reads + v0, kChunk, width, d.dv, (long long)kChunk * d.dv);
    load_planes<NV>(S, ldv, planeS, states + v0, d.dk, width, d.dv, planeG);
    copies_done();
    __syncthreads();
    product<2, NV, false, true, kParts<I>, 2>(dp, tO, m0, tW, p0);
    product<2, NV, false, true, 2, 2>(dl, tR, m0, tW, p0);
    product<kNP, NV, false, true, kParts<I>, 2>(dq, tO, m0, tS, n0);
    product<kNP, NV, false, true, 2, 2>(dk, tR, m0, tS, n0);
    {  // a quarter of a warp's lanes takes a token's columns: V' . dV and v . dv
      const int i = tid >> 2, sub = (tid & 3) * 8;
      float wr = 0.f, vr = 0.f;
      if (i < rows) {
        const I* v = head_at<I>(a.v, b, t0 + i, h) + v0;
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
          if (sub + k >= width) break;
          const float2 w = get2(W + i * ldv + sub + k, planeX), r = get2(R + i * ldv + sub + k, planeX);
          const float2 x = pair_of(v + sub + k, d.wide);
          wr += w.x * r.x + w.y * r.y;
          vr += x.x * r.x + x.y * r.y;
        }
      }
      wr += __shfl_xor_sync(0xffffffffu, wr, 1);
      vr += __shfl_xor_sync(0xffffffffu, vr, 1);
      wr += __shfl_xor_sync(0xffffffffu, wr, 2);
      vr += __shfl_xor_sync(0xffffffffu, vr, 2);
      if ((tid & 3) == 0) {
        dots[0][i] += wr;
        dots[1][i] += vr;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float2 x = G[m0 + g + k * 8];
    const float grown = expf(x.x + x.y);
#pragma unroll
    for (int n = 0; n < 2 * kNP; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        dk[n][2 * k + e] *= -grown;
        dq[n][2 * k + e] *= grown;
      }
  }
  // 2. What meets the gradient of the state after it: dK through the writes, and <dS', S'>.
  const bf16* dstates = a.dstates + at.n * 2 * d.dk * d.dv;
  float handed = 0.f;
  for (int v0 = 0; v0 < d.dv; v0 += NV) {
    const int width = min(NV, d.dv - v0);
    __syncthreads();
    load_planes<NV>(S, ldv, planeS, dstates + v0, d.dk, width, d.dv, planeG);
    for (int i = tid; i < kChunk * NV / 2; i += blockDim.x) {
      const int r = i / (NV / 2), col = i % (NV / 2) * 2;
      float2 w = make_float2(0.f, 0.f);
      if (col < width) w = get2(writes + r * d.dv + v0 + col, kChunk * d.dv);
      const float f = decay_between(G[kChunk - 1], G[r]);
      put2(W + r * ldv + col, planeX, w.x * f, w.y * f);
    }
    copies_done();
    __syncthreads();
    product<kNP, NV, false, true, 2, 2>(dk, tW, m0, tS, n0);
    for (int i = tid; i < d.dk * NV / 2; i += blockDim.x) {
      const int r = i / (NV / 2), col = i % (NV / 2) * 2;
      if (col >= width) continue;
      const bf16* after = states + 2 * planeG + r * d.dv + v0 + col;  // the next state's planes follow
      const float2 x = get2(S + r * ldv + col, planeS);
      const float2 y = make_float2(__bfloat162float(after[0]) + __bfloat162float(after[planeG]),
                                   __bfloat162float(after[1]) + __bfloat162float(after[planeG + 1]));
      handed += x.x * y.x + x.y * y.y;
    }
  }
  handed = lanes_sum(handed);
  if (lane == 0) state_dot[warp] = handed;
  __syncthreads();
  // 3. What meets the chunk's own tokens. dP D goes in with rq_i rk_j, dL D with rk_i rk_j, so that q and k stay as given.
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = m0 + g + (e / 2) * 8, j = p0 + n * 8 + t2 + (e & 1);
      const float w = j <= i ? decay_between(G[i], G[j]) * rk[j] : 0.f;
      const float p = dp[n][e] * w * rq[i], l = j < i ? -dl[n][e] * w * rk[i] : 0.f;
      const bf16 ph = __float2bfloat16_rn(p), lh = __float2bfloat16_rn(l);
      C[i * kLdC + j] = j <= i ? ph : __float2bfloat16_rn(0.f);
      C[planeC + i * kLdC + j] = j <= i ? __float2bfloat16_rn(p - __bfloat162float(ph)) : __float2bfloat16_rn(0.f);
      if (j > i) continue;
      const bf16 ll = __float2bfloat16_rn(l - __bfloat162float(lh));
      N[i * kLdC + j] = N[j * kLdC + i] = lh;
      N[planeC + i * kLdC + j] = N[planeC + j * kLdC + i] = ll;
    }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = m0 + g + k * 8;
#pragma unroll
    for (int n = 0; n < 2 * kNP; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        dq[n][2 * k + e] *= rq[i];
        dk[n][2 * k + e] *= rk[i];
      }
  }
  __syncthreads();
  product<kNP, kChunk, false, false, 2, kParts<I>>(dq, tC, m0, tK, n0);
  product<kNP, kChunk, true, false, 2, kParts<I>>(dk, tC, m0, tQ, n0);
  product<kNP, kChunk, false, false, 2, kParts<I>>(dk, tN, m0, tK, n0);
  // Now dq = rq dq^ and dk = rk dk^, of the scaled rows q^ and k^. q^ . dq^ = q . dq.
  float qd[2] = {0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int n = 0; n < 2 * kNP; ++n) {
      const int i = m0 + g + k * 8, col = n0 + n * 8 + t2;
      float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(Q + i * ldk + col));
      if (kParts<I> == 2) x = get2(Q + i * ldk + col, planeK);
      qd[k] += x.x * dq[n][2 * k] + x.y * dq[n][2 * k + 1];
    }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    qd[k] += __shfl_xor_sync(0xffffffffu, qd[k], 1);
    qd[k] += __shfl_xor_sync(0xffffffffu, qd[k], 2);
  }
  __syncthreads();
  float* half_dot = reinterpret_cast<float*>(N);  // two column halves of each row: added in order
  if ((lane & 3) == 0) {
    half_dot[(warp / 4) * kChunk + m0 + g] = qd[0];
    half_dot[(warp / 4) * kChunk + m0 + g + 8] = qd[1];
  }
  __syncthreads();
  if (tid < kChunk) dots[2][tid] = half_dot[tid] + half_dot[kChunk + tid];
  __syncthreads();
  if (warp == 0) {  // the gates: sums from each token to the chunk's end, two tokens a lane
    float after = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) after += state_dot[w];
    const float x = dots[2][2 * lane] - dots[1][2 * lane], y = dots[2][2 * lane + 1] - dots[1][2 * lane + 1];
    float sum = x + y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float up = __shfl_down_sync(0xffffffffu, sum, o);
      if (lane + o < 32) sum += up;
    }
    const float a_log = load_any(a.g.a_log, a.g.a_log_type, h), dt = load_any(a.g.dt_bias, a.g.dt_bias_type, h);
    double sum_log = 0.0, sum_bias = 0.0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = 2 * lane + k;
      if (i >= rows) continue;
      const Gate gate = gate_of(ElemOf<I>::up(*head_at<I>(a.g.a, b, t0 + i, h)), a_log, dt);
      // Nothing passes a gate whose factor is 0 in fp32: what the sum holds then is its rounding.
      const float dg = gate.log_decay < -104.f ? 0.f : (k ? sum - x : sum) + after;
      const float da = -dg * gate.rate * gate.slope;
      const float beta = a.keep.beta[at.n * kChunk + i];
      const float db = beta > 1e-20f ? (1.f - beta) * (dots[0][i] / beta) : 0.f;  // V' = beta E; below, db is under 1e-20 dV . E
      const long long to = ((long long)b * d.T + t0 + i) * d.H + h;
      reinterpret_cast<I*>(a.da)[to] = ElemOf<I>::down(da);
      reinterpret_cast<I*>(a.db)[to] = ElemOf<I>::down(db);
      sum_log += (double)dg * gate.log_decay;
      sum_bias += da;
    }
    sum_log = lanes_sum(sum_log);
    sum_bias = lanes_sum(sum_bias);
    if (lane == 0) {
      a.part[at.n * 2] = (float)sum_log;
      a.part[at.n * 2 + 1] = (float)sum_bias;
    }
  }
  // 4. Sums over the key head's value heads, then back through the rows' scaling: with x a row, r its reciprocal length and
  // y = r d / (scaled row): dx = y - x r^2 (x . y).
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int n = 0; n < 2 * kNP; ++n) {
      const int i = m0 + g + k * 8, col = n0 + n * 8 + t2;
      // Q and K lie under F: the rows are read again from global memory below
      *reinterpret_cast<float2*>(F + i * ldF + col) = make_float2(dq[n][2 * k], dq[n][2 * k + 1]);
      *reinterpret_cast<float2*>(F + (kChunk + i) * ldF + col) = make_float2(dk[n][2 * k], dk[n][2 * k + 1]);
    }
  cg::cluster_group cluster = cg::this_cluster();
  if (group > 1) cluster.sync();
  else __syncthreads();
  // The rows of both are shared out over the cluster's warps.
  for (int r = hg * 8 + warp; r < 2 * kChunk; r += 8 * group) {
    const int i = r % kChunk;
    if (i >= rows) continue;
    const bool of_k = r >= kChunk;
    const I* x = of_k ? head_at<I>(a.k, b, t0 + i, hk) : head_at<I>(a.q, b, t0 + i, hk);
    float y[DK / 32], v[DK / 32], dot = 0.f;
#pragma unroll
    for (int k = 0; k < DK / 32; ++k) {
      const int col = k * 32 + lane;
      y[k] = 0.f;
      for (int o = 0; o < group; ++o) {
        const float* f = group > 1 ? cluster.map_shared_rank(F, o) : F;
        y[k] += f[r * ldF + col];
      }
      v[k] = col < d.dk ? ElemOf<I>::up(x[col]) : 0.f;
      dot = fmaf(v[k], y[k], dot);
    }
    dot = lanes_sum(dot);
    const float len = of_k ? rk[i] : rq[i] / d.scale;
    I* to = reinterpret_cast<I*>(of_k ? a.dk : a.dq) + (((long long)b * d.T + t0 + i) * d.Hk + hk) * d.dk;
#pragma unroll
    for (int k = 0; k < DK / 32; ++k) {
      const int col = k * 32 + lane;
      if (col < d.dk) to[col] = ElemOf<I>::down(y[k] - v[k] * (len * len * dot));
    }
  }
  if (group > 1) cluster.sync();  // no CTA leaves while its rows are read
}

// The chunks' sums for a_log and dt_bias of one head, in a fixed order.
__global__ void __launch_bounds__(256) gates_kernel(const DeltaBwd a) {
  __shared__ double red[2][8];
  const DeltaDims& d = a.d;
  const int h = blockIdx.x;
  double s[2] = {0.0, 0.0};
  for (long long i = threadIdx.x; i < (long long)d.B * d.chunks; i += blockDim.x) {
    const long long n = (i / d.chunks * d.H + h) * d.chunks + i % d.chunks;
    s[0] += a.part[2 * n];
    s[1] += a.part[2 * n + 1];
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    s[k] = lanes_sum(s[k]);
    if ((threadIdx.x & 31) == 0) red[k][threadIdx.x >> 5] = s[k];
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    double t = 0.0;
    for (int w = 0; w < 8; ++w) t += red[threadIdx.x][w];
    if (threadIdx.x == 0) store_any(a.da_log, a.g.a_log_type, h, (float)t);
    else store_any(a.ddt_bias, a.g.dt_bias_type, h, (float)t);
  }
}

// ---------------------------------------------------------------- launches
template <typename F>
void allow(F* kernel, size_t bytes) {
  cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

template <typename I, int DK>
int fwd(const DeltaFwd& a, cudaStream_t s) {
  constexpr int P = kParts<I>, NV = 64;
  const DeltaDims& d = a.d;
  const unsigned heads = (unsigned)(d.B * d.H), slices = (d.dv + NV - 1) / NV;
  const size_t rows = sizeof(bf16) * kChunk * (DK + kPad) * P, tokens = sizeof(bf16) * 2 * kChunk * (NV + kPad),
               state = sizeof(bf16) * 2 * DK * (NV + kPad), square = sizeof(bf16) * 2 * kChunk * kLdC;
  if (d.chunks > 0) {
    const size_t bytes = 2 * rows + sizeof(float) * kChunk * (kChunk + 4);
    allow(prepare_kernel<I, DK>, bytes);
    prepare_kernel<I, DK><<<heads * d.chunks, 128, bytes, s>>>(a);
  }
  const size_t bytes = rows + tokens + state + square;
  allow(state_kernel<I, DK, NV>, bytes);
  state_kernel<I, DK, NV><<<heads * slices, 256, bytes, s>>>(a);
  if (d.chunks == 0) return 1;
  allow(output_kernel<I, DK, NV>, bytes);
  output_kernel<I, DK, NV><<<heads * d.chunks * slices, 256, bytes, s>>>(a);
  return 3;
}

template <typename I, int DK>
int bwd(const DeltaBwd& a, cudaStream_t s) {
  constexpr int P = kParts<I>, NV = 64, NI = 32;
  const DeltaDims& d = a.d;
  const unsigned heads = (unsigned)(d.B * d.H);
  const size_t rows = sizeof(bf16) * kChunk * (DK + kPad) * P;
  if (heads > 0) {
    constexpr int V = kParts<I> == 1 ? NV : 32;  // two parts of q, k and dO leave room for 32 columns
    const size_t tokens = sizeof(bf16) * kChunk * (V + kPad), state = sizeof(bf16) * 2 * DK * (V + kPad),
                 square = sizeof(bf16) * 2 * kChunk * kLdC;
    const size_t bytes = 2 * rows + (P + 4) * tokens + state + 2 * square;
    allow(dstate_kernel<I, DK, V>, bytes);
    dstate_kernel<I, DK, V><<<heads * ((d.dv + V - 1) / V), 256, bytes, s>>>(a);
  }
  if (heads * d.chunks > 0) {
    const size_t slice = sizeof(bf16) * ((P + 4) * kChunk * (NI + kPad) + 2 * DK * (NI + kPad)),
                 squares = sizeof(bf16) * 4 * kChunk * kLdC, sums = sizeof(float) * 2 * kChunk * (DK + 4);
    size_t bytes = 2 * rows + (slice > squares ? slice : squares);
    if (bytes < sums) bytes = sums;
    allow(inputs_kernel<I, DK>, bytes);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(heads * d.chunks);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = d.H / d.Hk;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, inputs_kernel<I, DK>, a);
  }
  gates_kernel<<<d.H, 256, 0, s>>>(a);
  return d.chunks > 0 ? 3 : 2;
}

}  // namespace

int delta_rule_fwd(const DeltaFwd& a, cudaStream_t s) {
  if (a.d.B * a.d.H == 0) return 0;
  if (a.d.type == Elem::kBF16) return a.d.dk <= 64 ? fwd<bf16, 64>(a, s) : fwd<bf16, 128>(a, s);
  return a.d.dk <= 64 ? fwd<__half, 64>(a, s) : fwd<__half, 128>(a, s);
}

int delta_rule_bwd(const DeltaBwd& a, cudaStream_t s) {
  if (a.d.H == 0) return 0;
  if (a.d.type == Elem::kBF16) return a.d.dk <= 64 ? bwd<bf16, 64>(a, s) : bwd<bf16, 128>(a, s);
  return a.d.dk <= 64 ? bwd<__half, 64>(a, s) : bwd<__half, 128>(a, s);
}

}  // namespace bw
