// Gated delta rule, token by token: for every sequence and value head, with u and w the rows of q and k scaled to length
// one (q also by the softmax-like scale),
//     S <- exp(g) S,   e = beta (v - S^T w),   S <- S + w e^T,   o = S^T u,
// S (dk, dv) in fp32, read and written once for all tokens of the call. Columns of S are independent: a CTA takes 32 of
// them, a thread 4 neighbouring ones of every 32nd row, so that S lies in registers and memory is moved in 128-byte
// rows of 16-byte accesses. Sums over rows: four lanes by shuffles, eight warps through shared memory.
//
// What bounds it: memory, 8 bytes of state for each element; with few sequences, the latency of one load, two sums and
// one store.
#include "delta_common.cuh"

namespace bw {
namespace {

constexpr int kCols = 32, kThreads = 256, kRowsOf = kMostKeyDim / 32;  // rows of a thread at most

template <typename I>
__global__ void __launch_bounds__(kThreads, 4) step_kernel(const DeltaStep s) {
  __shared__ float rows[2][kMostKeyDim];  // q, k
  __shared__ float part[2][8][kCols];
  __shared__ float norm[2];
  const DeltaDims& d = s.d;
  const int slices = (d.dv + kCols - 1) / kCols;
  const int slice = blockIdx.x % slices;
  const long long bh = blockIdx.x / slices;
  const int b = (int)(bh / d.H), h = (int)(bh % d.H), hk = h / (d.H / d.Hk);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = slice * kCols + (lane & 7) * 4;       // of the thread's four columns
  const int row0 = warp * 4 + (lane >> 3);              // its rows: row0 + 32 i
  const bool in = col < d.dv;
  float* base = s.state + b * s.ssb + h * s.ssh + col;
  float4 S[kRowsOf];
#pragma unroll
  for (int i = 0; i < kRowsOf; ++i) {
    const int r = row0 + 32 * i;
    S[i] = in && r < d.dk ? *reinterpret_cast<const float4*>(base + (long long)r * d.dv) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const float a_log = load_any(s.g.a_log, s.g.a_log_type, h), dt = load_any(s.g.dt_bias, s.g.dt_bias_type, h);
  const I *qp = reinterpret_cast<const I*>(s.q.p) + b * s.q.sb + hk * s.q.sh, *kp = reinterpret_cast<const I*>(s.k.p) + b * s.k.sb + hk * s.k.sh;
  const I* vp = reinterpret_cast<const I*>(s.v.p) + b * s.v.sb + h * s.v.sh;
  const I *ap = reinterpret_cast<const I*>(s.g.a.p) + b * s.g.a.sb + h * s.g.a.sh, *bp = reinterpret_cast<const I*>(s.g.b.p) + b * s.g.b.sb + h * s.g.b.sh;
  I* out = reinterpret_cast<I*>(s.out) + ((long long)b * d.T * d.H + h) * d.dv;
  for (int t = 0; t < d.T; ++t) {
    if (warp < 2) {
      const I* x = (warp == 0 ? qp + t * s.q.st : kp + t * s.k.st);
      float sq = 0.f;
      for (int i = lane; i < kMostKeyDim; i += 32) {
        const float v = i < d.dk ? ElemOf<I>::up(x[i]) : 0.f;
        rows[warp][i] = v;
        sq = fmaf(v, v, sq);
      }
      sq = lanes_sum(sq);
      if (lane == 0) norm[warp] = rsqrtf(sq + 1e-6f) * (warp == 0 ? d.scale : 1.f);
    }
    const Gate gate = gate_of(ElemOf<I>::up(ap[t * s.g.a.st]), a_log, dt);
    const float decay = expf(gate.log_decay), beta = sigmoid(ElemOf<I>::up(bp[t * s.g.b.st]));
    float v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = in ? ElemOf<I>::up(vp[t * s.v.st + col + c]) : 0.f;
    __syncthreads();
    const float rq = norm[0], rk = norm[1];
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float w[kRowsOf];
#pragma unroll
    for (int i = 0; i < kRowsOf; ++i) {
      w[i] = rows[1][row0 + 32 * i] * rk;
      S[i].x *= decay;
      S[i].y *= decay;
      S[i].z *= decay;
      S[i].w *= decay;
      sum.x = fmaf(S[i].x, w[i], sum.x);
      sum.y = fmaf(S[i].y, w[i], sum.y);
      sum.z = fmaf(S[i].z, w[i], sum.z);
      sum.w = fmaf(S[i].w, w[i], sum.w);
    }
    const auto total = [&](float4 x, int which) {
#pragma unroll
      for (int o = 8; o < 32; o <<= 1) {
        x.x += __shfl_xor_sync(0xffffffffu, x.x, o);
        x.y += __shfl_xor_sync(0xffffffffu, x.y, o);
        x.z += __shfl_xor_sync(0xffffffffu, x.z, o);
        x.w += __shfl_xor_sync(0xffffffffu, x.w, o);
      }
      if (lane < 8) *reinterpret_cast<float4*>(&part[which][warp][lane * 4]) = x;
    };
    total(sum, 0);
    __syncthreads();
    float e[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int o = 0; o < 8; ++o) {
      const float4 x = *reinterpret_cast<const float4*>(&part[0][o][(lane & 7) * 4]);
      e[0] += x.x;
      e[1] += x.y;
      e[2] += x.z;
      e[3] += x.w;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) e[c] = beta * (v[c] - e[c]);
    sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kRowsOf; ++i) {
      const float u = rows[0][row0 + 32 * i] * rq;
      S[i].x = fmaf(w[i], e[0], S[i].x);
      S[i].y = fmaf(w[i], e[1], S[i].y);
      S[i].z = fmaf(w[i], e[2], S[i].z);
      S[i].w = fmaf(w[i], e[3], S[i].w);
      sum.x = fmaf(S[i].x, u, sum.x);
      sum.y = fmaf(S[i].y, u, sum.y);
      sum.z = fmaf(S[i].z, u, sum.z);
      sum.w = fmaf(S[i].w, u, sum.w);
    }
    total(sum, 1);
    __syncthreads();
    if (warp == 0 && slice * kCols + lane < d.dv) {
      float o = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) o += part[1][k][lane];
      out[(long long)t * d.H * d.dv + slice * kCols + lane] = ElemOf<I>::down(o);
    }
  }
#pragma unroll
  for (int i = 0; i < kRowsOf; ++i) {
    const int r = row0 + 32 * i;
    if (in && r < d.dk) *reinterpret_cast<float4*>(base + (long long)r * d.dv) = S[i];
  }
}

}  // namespace

void delta_step(const DeltaStep& s, cudaStream_t stream) {
  const long long grid = (long long)s.d.B * s.d.H * ((s.d.dv + kCols - 1) / kCols);
  if (grid == 0 || s.d.T == 0) return;
  if (s.d.type == Elem::kBF16) step_kernel<__nv_bfloat16><<<(unsigned)grid, kThreads, 0, stream>>>(s);
  else if (s.d.type == Elem::kF16) step_kernel<__half><<<(unsigned)grid, kThreads, 0, stream>>>(s);
  else step_kernel<float><<<(unsigned)grid, kThreads, 0, stream>>>(s);
}

}  // namespace bw
