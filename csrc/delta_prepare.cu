// Gated delta rule in chunks: what each chunk has by itself (gates, lengths, P and the inverse). delta_state.cu says what it is for.
//
// 4 warps to a chunk of a value head; K K^T and Q K^T on 16-bit tensor instructions of a warp, since a product of 64 x 64 x 128
// is over before a tensor-memory pipeline has begun.
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

struct Place3 {
  int b, h, c;
  long long bh, n;
  __device__ Place3(const DeltaDims& d, long long head, int chunk) : c(chunk), bh(head), n(head * d.chunks + chunk) {
    b = (int)(head / d.H);
    h = (int)(head % d.H);
  }
};

// ---------------------------------------------------------------- prepare
// One chunk of one value head: 4 warps, 16 tokens' rows of both products each. The inverse of I + A, A strictly lower: the two
// diagonal blocks of 32 by forward substitution, a column to each of 64 threads, then the block below them as
// -T22 A21 T11 by all; all in fp32.
template <typename I, int DK>
__global__ void __launch_bounds__(128) prepare_kernel(const DeltaFwd a) {
  constexpr int ld = DK + kPad, plane = kChunk * ld, ldA = kChunk + 4, ldU = 36;
  extern __shared__ __align__(16) unsigned char raw[];
  bf16* Q = reinterpret_cast<bf16*>(raw);
  bf16* K = Q + kParts<I> * plane;
  float* A = reinterpret_cast<float*>(K + kParts<I> * plane);  // (64, ldA): L diag(beta), then the inverse
  float* U = A + kChunk * ldA;                                 // (32, ldU): A21 T11
  __shared__ float2 G[kChunk];
  __shared__ float beta[kChunk], rk[kChunk], rq[kChunk], logs[kChunk];
  const DeltaDims& d = a.d;
  const Place3 at(d, blockIdx.x / d.chunks, blockIdx.x % d.chunks);
  const int group = d.H / d.Hk, hk = at.h / group;
  const int t0 = at.c * kChunk, rows = min(kChunk, d.T - t0);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long m = ((long long)at.b * d.Hk + hk) * d.chunks + at.c;
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
  {  // lengths: a row of k or q to each thread
    const bf16* x = (tid < kChunk ? K : Q) + (tid & 63) * ld;
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
    const float len = rsqrtf(sq[0] + sq[1] + 1e-6f);
    if (tid < kChunk) rk[tid] = len;
    else rq[tid - kChunk] = len * d.scale;
  }
  float kk[8][4], qk[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) kk[i][j] = qk[i][j] = 0.f;
  const Tile tk{K, ld, plane}, tq{Q, ld, plane};
  product<4, DK, false, true, kParts<I>, kParts<I>>(kk, tk, warp * 16, tk, 0, warp + 1);
  product<4, DK, false, true, kParts<I>, kParts<I>>(qk, tq, warp * 16, tk, 0, warp + 1);
  __syncthreads();
  if (at.h % group == 0) {  // the rows as tiles, for the other kernels
    if (tid < kChunk) {
      a.keep.rk[m * kChunk + tid] = rk[tid];
      a.keep.rq[m * kChunk + tid] = rq[tid];
    }
    constexpr int kV = DK / 8;
    for (int i = tid; i < 2 * kParts<I> * kChunk * kV; i += 128) {
      const int which = i / (kParts<I> * kChunk * kV), part = i / (kChunk * kV) % kParts<I>, r = i / kV % kChunk, c = i % kV;
      unsigned char* to = (which ? a.keep.keys : a.keep.queries) + (m * kParts<I> + part) * (DK / 64) * kTok;
      *reinterpret_cast<uint4*>(to + (c >> 3) * kTok + piece_at(r, c & 7)) =
          *reinterpret_cast<const uint4*>((which ? K : Q) + part * plane + r * ld + c * 8);
    }
  }
  unsigned char* P = a.keep.attend + at.n * 2 * kTok;
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
      uint32_t hi, lo;
      halves(p[0], p[1], hi, lo);
      *reinterpret_cast<uint32_t*>(P + element_at(i, j, 0)) = hi;
      *reinterpret_cast<uint32_t*>(P + kTok + element_at(i, j, 0)) = lo;
      *reinterpret_cast<float2*>(A + i * ldA + j) = make_float2(l[0], l[1]);
    }
  __syncthreads();
  float x[32];
  const int block = (tid >> 5) * 32, col = tid & 31;
  if (tid < kChunk) {  // x_i = [i = column] - sum_{m < i} A_im x_m
    const float* B = A + block * ldA + block;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      float s[4] = {i == col ? 1.f : 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < i; ++k) s[k & 3] = fmaf(-B[i * ldA + k], x[k], s[k & 3]);
      x[i] = (s[0] + s[1]) + (s[2] + s[3]);
    }
    __syncwarp();  // the block belongs to this warp
#pragma unroll
    for (int i = 0; i < 32; ++i) A[(block + i) * ldA + block + col] = x[i];
  }
  __syncthreads();
  const int row = tid >> 2, c8 = (tid & 3) * 8;
  const auto rows_times = [&](const float* X, const float* Y, int ldY, float (&s)[8]) {  // (row of X) Y, 32 terms
#pragma unroll
    for (int k = 0; k < 8; ++k) s[k] = 0.f;
#pragma unroll 8
    for (int k = 0; k < 32; ++k) {
      const float f = X[row * ldA + k];
      const float4 y0 = *reinterpret_cast<const float4*>(Y + k * ldY + c8), y1 = *reinterpret_cast<const float4*>(Y + k * ldY + c8 + 4);
      s[0] = fmaf(f, y0.x, s[0]);
      s[1] = fmaf(f, y0.y, s[1]);
      s[2] = fmaf(f, y0.z, s[2]);
      s[3] = fmaf(f, y0.w, s[3]);
      s[4] = fmaf(f, y1.x, s[4]);
      s[5] = fmaf(f, y1.y, s[5]);
      s[6] = fmaf(f, y1.z, s[6]);
      s[7] = fmaf(f, y1.w, s[7]);
    }
  };
  float s[8];
  rows_times(A + 32 * ldA, A, ldA, s);
  *reinterpret_cast<float4*>(U + row * ldU + c8) = make_float4(s[0], s[1], s[2], s[3]);
  *reinterpret_cast<float4*>(U + row * ldU + c8 + 4) = make_float4(s[4], s[5], s[6], s[7]);
  __syncthreads();
  rows_times(A + 32 * ldA + 32, U, ldU, s);
  *reinterpret_cast<float4*>(A + (32 + row) * ldA + c8) = make_float4(-s[0], -s[1], -s[2], -s[3]);
  *reinterpret_cast<float4*>(A + (32 + row) * ldA + c8 + 4) = make_float4(-s[4], -s[5], -s[6], -s[7]);
  __syncthreads();
  unsigned char* T = a.keep.solve + at.n * 2 * kTok;
  for (int i = tid; i < kChunk * 8; i += 128) {
    const int r = i >> 3, p = i & 7;
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = p * 8 + k <= r ? A[r * ldA + p * 8 + k] : 0.f;
    put8(T + piece_at(r, p), T + kTok + piece_at(r, p), f);
  }
}

template <typename I, int DK>
void prepare(const DeltaFwd& a, cudaStream_t s) {
  const size_t bytes = 2 * kParts<I> * sizeof(bf16) * kChunk * (DK + kPad) + sizeof(float) * (kChunk * (kChunk + 4) + 32 * 36);
  cudaFuncSetAttribute(prepare_kernel<I, DK>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  prepare_kernel<I, DK><<<(unsigned)(a.d.B * a.d.H) * a.d.chunks, 128, bytes, s>>>(a);
}

}  // namespace

void delta_prepare(const DeltaFwd& a, cudaStream_t s) {
  if (a.d.type == Elem::kBF16) return a.d.dk <= 64 ? prepare<bf16, 64>(a, s) : prepare<bf16, 128>(a, s);
  return a.d.dk <= 64 ? prepare<__half, 64>(a, s) : prepare<__half, 128>(a, s);
}

}  // namespace bw
