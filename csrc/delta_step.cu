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
#include "tc_common.cuh"

namespace bw {
namespace {

constexpr int kCols = 32, kThreads = 256, kRowsOf = kMostKeyDim / 32;  // rows of a thread at most

template <typename I>
__global__ void __launch_bounds__(kThreads, 4) step_kernel(const DeltaStep s) {
  __shared__ float rows[2][kMostKeyDim];  // q, k
  __shared__ __align__(16) float part[2][8][kCols];
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

// Many sequences: CTAs that stay and take head after head, the states of the next ones on their way by bulk copies while one is
// worked on in registers and another goes back. A thread takes four neighbouring columns of every 16th row; sums over rows go by
// shuffles over four of them, then through shared memory. 2,048 heads of 128 x 128: 62 us, 4.3 TB/s. What bounds it: one group of
// threads takes a head's waits, its two sums and its way back one behind the other, 4.5 us a head; the bytes would take 41 us.
constexpr int kStayThreads = 512, kStayRows = kMostKeyDim / 16, kBuffers = 3, kStayCols = 128,
              kStayFloats = kMostKeyDim * kStayCols;

struct StayShared {
  uint64_t full[kBuffers];
  float rows[2][2][kMostKeyDim];  // q and k, of this token and of the next one
  float norm[2][2];
  alignas(16) float part[2][4][kStayCols];
};

template <typename I>
__global__ void __launch_bounds__(kStayThreads, 1) step_stay_kernel(const DeltaStep s) {
  extern __shared__ __align__(128) unsigned char mem[];
  float* const states = reinterpret_cast<float*>(mem);
  StayShared& sh = *reinterpret_cast<StayShared*>(mem + kBuffers * kStayFloats * 4);
  const DeltaDims& d = s.d;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int heads = d.B * d.H, by = gridDim.x, bytes = d.dk * d.dv * 4;
  const int col = (warp & 3) * 32 + (lane & 7) * 4, row0 = (warp >> 2) * 4 + (lane >> 3);
  const bool in = col < d.dv;
  const auto state_of = [&](int head) { return s.state + head / d.H * s.ssb + head % d.H * s.ssh; };
  const auto load = [&](int head, int buffer) {
    mbar_arrive_expect_tx(&sh.full[buffer], bytes);
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(states + buffer * kStayFloats)),
                 "l"(state_of(head)), "r"(bytes), "r"(smem_u32(&sh.full[buffer]))
                 : "memory");
  };
  if (tid == 0) {
    for (int i = 0; i < kBuffers; ++i) mbar_init(&sh.full[i], 1);
    fence_barrier_init();
    fence_proxy_async_smem();
    for (int i = 0; i < kBuffers - 1; ++i)
      if ((int)blockIdx.x + i * by < heads) load(blockIdx.x + i * by, i);
  }
  // The row of q or k of token t: the first two warps bring it, with its length.
  const auto fetch = [&](int head, int t, float (&x)[kMostKeyDim / 32]) {
    const int b = head / d.H, hk = head % d.H / (d.H / d.Hk);
    const I* from = warp == 0 ? reinterpret_cast<const I*>(s.q.p) + b * s.q.sb + hk * s.q.sh + t * s.q.st
                              : reinterpret_cast<const I*>(s.k.p) + b * s.k.sb + hk * s.k.sh + t * s.k.st;
#pragma unroll
    for (int i = 0; i < kMostKeyDim / 32; ++i) x[i] = i * 32 + lane < d.dk ? ElemOf<I>::up(from[i * 32 + lane]) : 0.f;
  };
  const auto place = [&](const float (&x)[kMostKeyDim / 32], int flip) {
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < kMostKeyDim / 32; ++i) {
      sh.rows[flip][warp][i * 32 + lane] = x[i];
      sq = fmaf(x[i], x[i], sq);
    }
    sq = lanes_sum(sq);
    if (lane == 0) sh.norm[flip][warp] = rsqrtf(sq + 1e-6f) * (warp == 0 ? d.scale : 1.f);
  };
  struct Token {
    float a, b, a_log, dt, v[4];
  };
  const auto read = [&](int head, int t, Token& x) {
    const int b = head / d.H, h = head % d.H;
    x.a = ElemOf<I>::up(reinterpret_cast<const I*>(s.g.a.p)[b * s.g.a.sb + h * s.g.a.sh + t * s.g.a.st]);
    x.b = ElemOf<I>::up(reinterpret_cast<const I*>(s.g.b.p)[b * s.g.b.sb + h * s.g.b.sh + t * s.g.b.st]);
    x.a_log = load_any(s.g.a_log, s.g.a_log_type, h);
    x.dt = load_any(s.g.dt_bias, s.g.dt_bias_type, h);
    const I* v = reinterpret_cast<const I*>(s.v.p) + b * s.v.sb + h * s.v.sh + t * s.v.st + col;
#pragma unroll
    for (int c = 0; c < 4; ++c) x.v[c] = in ? ElemOf<I>::up(v[c]) : 0.f;
  };
  const auto total = [&](float4 x, int which) {
#pragma unroll
    for (int o = 8; o < 32; o <<= 1) {
      x.x += __shfl_xor_sync(0xffffffffu, x.x, o);
      x.y += __shfl_xor_sync(0xffffffffu, x.y, o);
      x.z += __shfl_xor_sync(0xffffffffu, x.z, o);
      x.w += __shfl_xor_sync(0xffffffffu, x.w, o);
    }
    if (lane < 8) *reinterpret_cast<float4*>(&sh.part[which][warp >> 2][col]) = x;
  };
  int head = blockIdx.x, flip = 0;
  float row[kMostKeyDim / 32];
  Token now, next;
  if (head < heads) {
    if (warp < 2) {
      fetch(head, 0, row);
      place(row, 0);
    }
    read(head, 0, now);
  }
  __syncthreads();
  bool dead = false;
  for (int n = 0; head < heads; ++n, head += by) {
    const int buffer = n % kBuffers;
    if (!mbar_wait(&sh.full[buffer], n / kBuffers & 1, s.err, kErrWaitFull)) dead = true;
    if (__syncthreads_or(dead)) break;
    float* S0 = states + buffer * kStayFloats + col;
    float4 S[kStayRows];
#pragma unroll
    for (int i = 0; i < kStayRows; ++i) {
      const int r = row0 + i * 16;
      S[i] = in && r < d.dk ? *reinterpret_cast<const float4*>(S0 + r * d.dv) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int t = 0; t < d.T; ++t) {
      const bool last = t + 1 == d.T;
      const int nh = last ? head + by : head, nt = last ? 0 : t + 1;
      if (nh < heads) {  // the next token's rows and gates, while this one is worked on
        if (warp < 2) fetch(nh, nt, row);
        read(nh, nt, next);
      }
      const Gate gate = gate_of(now.a, now.a_log, now.dt);
      const float decay = expf(gate.log_decay), beta = sigmoid(now.b);
      const float rq = sh.norm[flip][0], rk = sh.norm[flip][1];
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      float w[kStayRows];
#pragma unroll
      for (int i = 0; i < kStayRows; ++i) {
        w[i] = sh.rows[flip][1][row0 + i * 16] * rk;
        S[i].x *= decay;
        S[i].y *= decay;
        S[i].z *= decay;
        S[i].w *= decay;
        sum.x = fmaf(S[i].x, w[i], sum.x);
        sum.y = fmaf(S[i].y, w[i], sum.y);
        sum.z = fmaf(S[i].z, w[i], sum.z);
        sum.w = fmaf(S[i].w, w[i], sum.w);
      }
      total(sum, 0);
      __syncthreads();
      float e[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int o = 0; o < 4; ++o) {
        const float4 x = *reinterpret_cast<const float4*>(&sh.part[0][o][col]);
        e[0] += x.x;
        e[1] += x.y;
        e[2] += x.z;
        e[3] += x.w;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) e[c] = beta * (now.v[c] - e[c]);
      sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kStayRows; ++i) {
        const float u = sh.rows[flip][0][row0 + i * 16] * rq;
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
      if (last) {
#pragma unroll
        for (int i = 0; i < kStayRows; ++i) {
          const int r = row0 + i * 16;
          if (in && r < d.dk) *reinterpret_cast<float4*>(S0 + r * d.dv) = S[i];
        }
        fence_proxy_async_smem();
      }
      if (warp < 2 && nh < heads) place(row, flip ^ 1);
      __syncthreads();
      if (last && tid == 0) {
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(state_of(head)),
                     "r"(smem_u32(states + buffer * kStayFloats)), "r"(bytes)
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        // The buffer before this one has been copied out: the head after the next one takes it.
        asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        if (head + (kBuffers - 1) * by < heads) load(head + (kBuffers - 1) * by, (n + kBuffers - 1) % kBuffers);
      }
      if (tid >= 128 && tid < 128 + d.dv) {
        float o = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) o += sh.part[1][k][tid - 128];
        const int b = head / d.H, h = head % d.H;
        reinterpret_cast<I*>(s.out)[(((long long)b * d.T + t) * d.H + h) * d.dv + tid - 128] = ElemOf<I>::down(o);
      }
      now = next;
      flip ^= 1;
    }
  }
  if (tid == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

template <typename I>
void launch(const DeltaStep& s, cudaStream_t stream) {
  const long long heads = (long long)s.d.B * s.d.H;
  // The pipeline pays for wide heads from some three of them for each SM on, and is taken from two on, where it costs 8 % at most: calls
  // of few and of many more heads then give the same bits. Below, more and smaller CTAs pay, and so they do for heads of 96
  // columns or fewer, which leave a quarter of the staying threads or more without a column. bf16, us with staying CTAs
  // and with a CTA to each 32 columns: heads of 128 x 128, 32 of them 5.5 and 4.0, 160 10.8 and 9.3, 320 15.0 and 13.9, 512 19.6
  // and 20.5, 1,024 33 and 39, 2,048 62 and 81; of 32 x 128, 512 14.0 and 14.9, 2,048 43 and 53; of 128 x 112, 320 14.8 and 14.3,
  // 2,048 61 and 78; of 96 x 96, 320 13.2 and 10.6, 2,048 53 and 51; of 64 x 64, 320 11.0 and 7.7, 2,048 43 and 30.
  if (heads >= 2 * 148 && s.d.dv > 96 && s.d.dv <= kStayCols && heads < (1ll << 30)) {
    constexpr int bytes = kBuffers * kStayFloats * 4 + (int)sizeof(StayShared);
    static_assert(bytes <= 227 * 1024, "shared memory");
    cudaFuncSetAttribute(step_stay_kernel<I>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    step_stay_kernel<I><<<148, kStayThreads, bytes, stream>>>(s);
    return;
  }
  const long long grid = heads * ((s.d.dv + kCols - 1) / kCols);
  step_kernel<I><<<(unsigned)grid, kThreads, 0, stream>>>(s);
}

}  // namespace

void delta_step(const DeltaStep& s, cudaStream_t stream) {
  if (s.d.B * s.d.H == 0 || s.d.T == 0) return;
  if (s.d.type == Elem::kBF16) launch<__nv_bfloat16>(s, stream);
  else if (s.d.type == Elem::kF16) launch<__half>(s, stream);
  else launch<float>(s, stream);
}

}  // namespace bw
