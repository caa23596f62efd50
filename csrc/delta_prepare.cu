// Gated delta rule in chunks: what each chunk has by itself (gates, lengths, P and the inverse). delta_state.cu says what it is for.
//
// 4 warps to a chunk of a key head; K K^T and Q K^T once for its value heads, on 16-bit tensor instructions of a warp, since a
// product of 64 x 64 x 128 is over before a tensor-memory pipeline has begun; then two value heads at a time. The inverse goes by
// halves: of the diagonal blocks of 32 by substitution, one column a thread, below them -(lower) block (upper), in fp32.
//
// What bounds it: the substitution's chain and shared memory. 4 x 2048 tokens, 16 key and 32 value heads of 128: 106 us (157
// with a value head to each CTA); 0.37 GB to read and write, 56 us.
#include "delta_tiles.cuh"

namespace bw {
namespace {

constexpr int kPad = 8;  // elements behind each row in shared memory: eight rows then lie in different banks

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

// acc (16 x 16 NP) += A (16 x K, from row m0) B (K x 16 NP, from column n0) of a warp, of which only the first `some` blocks of
// 16 columns are wanted. kAT: A is stored (K, M); kBT: B is
// stored (N, K). kA and kB: parts of each.
template <int NP, int K, bool kAT, bool kBT, int kA, int kB>
__device__ __forceinline__ void product(float (&acc)[2 * NP][4], const Tile& A, int m0, const Tile& B, int n0, int some) {
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
      if (n >= some) break;
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

__device__ __forceinline__ void put2(bf16* p, int lo, float x, float y) {
  uint32_t h, l;
  halves(x, y, h, l);
  *reinterpret_cast<uint32_t*>(p) = h;
  *reinterpret_cast<uint32_t*>(p + lo) = l;
}

// ---------------------------------------------------------------- loads
__device__ __forceinline__ void copy16(bf16* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_at(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory"); }

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

// ---------------------------------------------------------------- prepare
// One chunk of one key head: 4 warps, 16 tokens' rows of both products each, which all its value heads share; those two at a time.
// The inverse of I + A, A strictly lower: the two diagonal blocks of 32 by forward substitution, a column to each thread
// of a warp, then the block below them as -T22 A21 T11; all in fp32.
template <typename I, int DK>
struct PrepareMem {
  static constexpr int ld = DK + kPad, plane = kChunk * ld, ldA = kChunk + 4, ldU = 36;
  static constexpr int kRowBytes = 2 * kParts<I> * plane * 2, kPairBytes = 2 * kChunk * ldA * 4;  // A lies where q and k were
  static constexpr int kFirst = kRowBytes > kPairBytes ? kRowBytes : kPairBytes, kBytes = kFirst + 2 * 32 * ldU * 4;
};

template <typename I, int DK>
__global__ void __launch_bounds__(128, kParts<I> == 1 ? 4 : 3) prepare_kernel(const DeltaFwd a) {
  using Mem = PrepareMem<I, DK>;
  constexpr int ld = Mem::ld, plane = Mem::plane, ldA = Mem::ldA, ldU = Mem::ldU;
  extern __shared__ __align__(16) unsigned char raw[];
  bf16* Q = reinterpret_cast<bf16*>(raw);
  bf16* K = Q + kParts<I> * plane;
  __shared__ float2 G[2][kChunk];
  __shared__ float beta[2][kChunk], rk[kChunk], rq[kChunk], logs[2][kChunk];
  const DeltaDims& d = a.d;
  const int group = d.H / d.Hk, c = blockIdx.x % d.chunks, b = blockIdx.x / d.chunks / d.Hk, hk = blockIdx.x / d.chunks % d.Hk;
  const int t0 = c * kChunk, rows = min(kChunk, d.T - t0);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, which = tid >> 6, tok = tid & 63;
  const long long m = blockIdx.x;  // (batch * Hk + key head) * chunks + chunk
  load_rows<I, DK>(Q, ld, plane, head_at<I>(a.q, b, t0, hk), a.q.st, rows, d.dk, d.wide);
  load_rows<I, DK>(K, ld, plane, head_at<I>(a.k, b, t0, hk), a.k.st, rows, d.dk, d.wide);
  copies_done();
  __syncthreads();
  {  // lengths: a row of k or q to each thread
    const bf16* x = (which ? Q : K) + tok * ld;
    float sq[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < DK; i += 8) {
      float f[8];
      raw_up<bf16>(*reinterpret_cast<const uint4*>(x + i), f);
      if (kParts<I> == 2) {
        float lo[8];
        raw_up<bf16>(*reinterpret_cast<const uint4*>(x + plane + i), lo);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] += lo[k];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) sq[k & 1] = fmaf(f[k], f[k], sq[k & 1]);
    }
    const float len = rsqrtf(sq[0] + sq[1] + 1e-6f) * (which ? d.scale : 1.f);
    (which ? rq : rk)[tok] = len;
    (which ? a.keep.rq : a.keep.rk)[m * kChunk + tok] = len;
  }
  // The rows as tiles, for the other kernels.
  constexpr int kV = DK / 8;
#pragma unroll 4
  for (int i = tid; i < 2 * kParts<I> * kChunk * kV; i += 128) {
    const int of_k = i / (kParts<I> * kChunk * kV), part = i / (kChunk * kV) % kParts<I>, r = i / kV % kChunk, p = i % kV;
    unsigned char* to = (of_k ? a.keep.keys : a.keep.queries) + (m * kParts<I> + part) * (DK / 64) * kTok;
    *reinterpret_cast<uint4*>(to + (p >> 3) * kTok + piece_at(r, p & 7)) =
        *reinterpret_cast<const uint4*>((of_k ? K : Q) + part * plane + r * ld + p * 8);
  }
  float kk[8][4], qk[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) kk[i][j] = qk[i][j] = 0.f;
  const Tile tk{K, ld, plane}, tq{Q, ld, plane};
  product<4, DK, false, true, kParts<I>, kParts<I>>(kk, tk, warp * 16, tk, 0, warp + 1);
  product<4, DK, false, true, kParts<I>, kParts<I>>(qk, tq, warp * 16, tk, 0, warp + 1);
  for (int g0 = 0; g0 < group; g0 += 2) {
    const int pair = min(2, group - g0);
    const long long n0 = ((long long)b * d.H + hk * group + g0) * d.chunks + c;  // the next value head is `chunks` further
    if (which < pair) {
      const int h = hk * group + g0 + which;
      float g = 0.f, w = 0.f;
      if (tok < rows) {
        g = gate_of(ElemOf<I>::up(*head_at<I>(a.g.a, b, t0 + tok, h)), load_any(a.g.a_log, a.g.a_log_type, h),
                    load_any(a.g.dt_bias, a.g.dt_bias_type, h)).log_decay;
        w = sigmoid(ElemOf<I>::up(*head_at<I>(a.g.b, b, t0 + tok, h)));
      }
      logs[which][tok] = g;
      beta[which][tok] = w;
      a.keep.beta[(n0 + which * d.chunks) * kChunk + tok] = w;
    }
    __syncthreads();  // q and k are read, too
    if (warp < pair) {  // sums of log-decays in 64 bits, kept as two floats
      const double x = logs[warp][2 * lane], y = logs[warp][2 * lane + 1];
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
        G[warp][2 * lane + k] = g;
        a.keep.total[(n0 + warp * d.chunks) * kChunk + 2 * lane + k] = g;
      }
    }
    __syncthreads();
    for (int e2 = 0; e2 < pair; ++e2) {
      unsigned char* P = a.keep.attend + (n0 + e2 * d.chunks) * 2 * kTok;
      float* A = reinterpret_cast<float*>(raw) + e2 * kChunk * ldA;  // L diag(beta), then the inverse
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const int i = warp * 16 + (lane >> 2) + (e ? 8 : 0);
        const float2 Gi = G[e2][i];
        const float qi = rq[i], ki = rk[i];
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const int j = n * 8 + (lane & 3) * 2;
          uint32_t hi = 0, lo = 0;
          float2 l = make_float2(0.f, 0.f);
          if (n < 2 * (warp + 1)) {  // else above the diagonal
            const float w0 = decay_between(Gi, G[e2][j]) * rk[j], w1 = decay_between(Gi, G[e2][j + 1]) * rk[j + 1];
            const float p0 = qk[n][e] * qi * w0, p1 = qk[n][e + 1] * qi * w1;
            const float l0 = kk[n][e] * ki * w0 * beta[e2][j], l1 = kk[n][e + 1] * ki * w1 * beta[e2][j + 1];
            halves(j <= i ? p0 : 0.f, j + 1 <= i ? p1 : 0.f, hi, lo);
            l = make_float2(j < i ? l0 : 0.f, j + 1 < i ? l1 : 0.f);
          }
          *reinterpret_cast<uint32_t*>(P + element_at(i, j, 0)) = hi;
          *reinterpret_cast<uint32_t*>(P + kTok + element_at(i, j, 0)) = lo;
          *reinterpret_cast<float2*>(A + i * ldA + j) = l;
        }
      }
    }
    __syncthreads();
    const int mine = warp >> 1;  // two warps to a head
    float* A = reinterpret_cast<float*>(raw) + mine * kChunk * ldA;
    float* U = reinterpret_cast<float*>(raw + Mem::kFirst) + mine * 32 * ldU;  // A21 T11
    const int block = (warp & 1) * 32;
    if (mine < pair) {  // x_i = [i = column] - sum_{m < i} A_im x_m
      const float* B = A + block * ldA + block;
      float x[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        float s[4] = {i == lane ? 1.f : 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < i; ++k) s[k & 3] = fmaf(-B[i * ldA + k], x[k], s[k & 3]);
        x[i] = (s[0] + s[1]) + (s[2] + s[3]);
      }
      __syncwarp();  // the block belongs to this warp
#pragma unroll
      for (int i = 0; i < 32; ++i) A[(block + i) * ldA + block + lane] = x[i];
    }
    __syncthreads();
    const int row = (warp & 1) * 16 + (lane >> 1), c16 = (lane & 1) * 16;
    const auto rows_times = [&](const float* X, const float* Y, int ldY, float (&s)[16]) {  // (row of X) Y, 32 terms
#pragma unroll
      for (int k = 0; k < 16; ++k) s[k] = 0.f;
#pragma unroll 4
      for (int k = 0; k < 32; ++k) {
        const float f = X[row * ldA + k];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 y = *reinterpret_cast<const float4*>(Y + k * ldY + c16 + 4 * e);
          s[4 * e] = fmaf(f, y.x, s[4 * e]);
          s[4 * e + 1] = fmaf(f, y.y, s[4 * e + 1]);
          s[4 * e + 2] = fmaf(f, y.z, s[4 * e + 2]);
          s[4 * e + 3] = fmaf(f, y.w, s[4 * e + 3]);
        }
      }
    };
    float s[16];
    if (mine < pair) {
      rows_times(A + 32 * ldA, A, ldA, s);
#pragma unroll
      for (int e = 0; e < 16; e += 4) *reinterpret_cast<float4*>(U + row * ldU + c16 + e) = make_float4(s[e], s[e + 1], s[e + 2], s[e + 3]);
    }
    __syncthreads();
    if (mine < pair) {
      rows_times(A + 32 * ldA + 32, U, ldU, s);
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<float4*>(A + (32 + row) * ldA + c16 + e) = make_float4(-s[e], -s[e + 1], -s[e + 2], -s[e + 3]);
    }
    __syncthreads();
    if (which < pair) {
      unsigned char* T = a.keep.solve + (n0 + which * d.chunks) * 2 * kTok;
      const float* X = reinterpret_cast<const float*>(raw) + which * kChunk * ldA;
#pragma unroll 4
      for (int i = tok; i < kChunk * 8; i += 64) {
        const int r = i >> 3, p = i & 7;
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = p * 8 + k <= r ? X[r * ldA + p * 8 + k] : 0.f;
        put8(T + piece_at(r, p), T + kTok + piece_at(r, p), f);
      }
    }
    __syncthreads();
  }
}

template <typename I, int DK>
void prepare(const DeltaFwd& a, cudaStream_t s) {
  constexpr int bytes = PrepareMem<I, DK>::kBytes;
  cudaFuncSetAttribute(prepare_kernel<I, DK>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  prepare_kernel<I, DK><<<(unsigned)(a.d.B * a.d.Hk) * a.d.chunks, 128, bytes, s>>>(a);
}

}  // namespace

void delta_prepare(const DeltaFwd& a, cudaStream_t s) {
  if (a.d.type == Elem::kBF16) return a.d.dk <= 64 ? prepare<bf16, 64>(a, s) : prepare<bf16, 128>(a, s);
  return a.d.dk <= 64 ? prepare<__half, 64>(a, s) : prepare<__half, 128>(a, s);
}

}  // namespace bw
