// Gated delta rule in chunks of 64 tokens, forward and backward.
//
// For each sequence and value head, with rows of k scaled to length one and rows of q to length `scale`:
//     S_t = exp(g_t) S_{t-1} + k_t beta_t (v_t - exp(g_t) S_{t-1}^T k_t)^T,      o_t = S_t^T q_t.
// Within a chunk let G_i be the sum of g from its start, D_ij = exp(G_i - G_j) for i >= j, L = strictly lower part of
// (K K^T) D, P = lower part of (Q K^T) D, S the state before the chunk and S' the one after it. Then
//     (I + L diag(beta)) E = V - diag(exp G) K S,     V' = diag(beta) E,
//     O = diag(exp G) Q S + P V',                     S' = exp(G_63) S + (diag(exp(G_63 - G)) K)^T V'.
// Kernels: `prepare` (every chunk by itself: lengths, decays, P and the inverse of the triangular matrix, in fp32), then `state`
// here (chunk after chunk: V', O and S').
//
// The backward goes the same way, from dO and dS':
//     dV' = P^T dO + diag(exp(G_63 - G)) K dS',       dV = (inverse)^T diag(beta) dV',
//     dS = exp(G_63) dS' + Q^T diag(exp G) dO - K^T diag(exp G) dV,                                    (`dstate`)
//     dP = lower(dO V'^T),  dL = -strictly lower(dV V'^T),
//     dQ = diag(exp G) dO S^T + (dP D) K,
//     dK = -diag(exp G) dV S^T + diag(exp(G_63 - G)) V' dS'^T + (dP D)^T Q + (dL D + (dL D)^T) K,
// and with b the logit of beta:  db_i = (1 - beta_i) dV_i . E_i. The log-decay's gradient at t is all that passes from before t to
// t or behind it: with M = dP P + dL L element by element and r the lengths' scaling left out,
//     dg_t = sum_{i >= t > j} M_ij + sum_{i >= t} exp(G_i) (q_i . S dO_i - k_i . S dV_i)
//          + sum_{j < t} exp(G_63 - G_j) k_j . dS' V'_j + exp(G_63) <dS', S>.                            (`inputs`)
// The same sum as the difference of what tokens take and give, q . dq - v . dv, needs fewer products, but its terms stay where a
// gate closes and what passes goes to nothing: half of a percent off over heads that keep e^-1 to e^-16 of a state.
//
// Matrix products run on 16-bit tensor instructions with fp32 sums. q, k and dO are bf16 as given, so they are exact; all
// that is computed (S, V', the inverse, P and their gradients) goes in as two bf16 halves, which keep 16 bits of 24: two products
// where one side is exact, three where both have halves (the product of the two low halves is below 2^-16 of the result).
// One half alone would round each operand by 2^-8, as much as the output's own rounding, several times over. fp16 inputs
// are two exact halves as well. The state itself stays in tensor memory in fp32 from the first chunk to the last; a final
// state is 1e-6 to 6e-6 of its norm off.
//
// Layout: a CTA has up to 128 value elements of a head, one a lane of tensor memory, so that all of a token's factors are by columns
// and the state's rows are the lanes: S^T, its reads by keys and queries, E and the outputs. One warp's first lane copies and
// multiplies, sixteen warps turn sums into halves, two compute the tokens' factors a chunk ahead.
//
// What bounds it: a chunk's chain of three products and three conversions, each waiting for the one before. 4 x 2048 tokens, 32
// heads of 128 x 128, bf16 (128 CTAs, 32 chunks each): state 152 us, dstate 165 us, 5 us a chunk, while the bytes (0.85
// GB each) would take 130 us. The first half of a state's columns is multiplied while the second is turned into halves. States are
// copied out behind the products that read them: in front of them, 156 and 181 us, since both read shared memory. On
// instructions of single warps (state and outputs as kernels of their own): 354 + 195 us and 594 us. With eight
// converting warps instead of sixteen a training pass took 8 % longer.
#include "delta_tiles.cuh"

namespace bw {
namespace {

// Beside the workers and the warp that copies and multiplies, two warps compute the next chunk's factors. With 64 of the workers,
// whose other warps then waited for them, a chunk took 1,700 of 10,200 cycles more.
constexpr int kThreads = kWorkers + 32 + kChunk;

// Of a chunk's tokens: what the products' columns are multiplied by.
struct Factors {
  float grown_k[kChunk];  // exp(G) rk
  float left_k[kChunk];   // exp(G_63 - G) rk
  float beta[kChunk];
  float left;             // exp(G_63)
};

// What they are made of, of one token: read a chunk ahead.
struct FactorParts {
  float2 G, end;
  float rk, rq, beta;
  __device__ __forceinline__ void read(const DeltaKept& keep, long long n, long long m, int i) {
    G = keep.total[n * kChunk + i];
    end = keep.total[n * kChunk + kChunk - 1];
    rk = keep.rk[m * kChunk + i];
    rq = keep.rq[m * kChunk + i];
    beta = keep.beta[n * kChunk + i];
  }
  __device__ __forceinline__ void fill(Factors& f, float* grown_q, int i) const {
    const float grown = __expf(G.x + G.y);
    f.grown_k[i] = grown * rk;
    grown_q[i] = grown * rq;
    f.left_k[i] = decay_between(end, G) * rk;
    f.beta[i] = beta;
    if (i == kChunk - 1) f.left = grown;
  }
};

template <typename I, int N>
__device__ __forceinline__ void put_column(I* p, long long st, int rows, const float (&x)[N]) {
  if (rows >= N) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      *p = ElemOf<I>::down(x[i]);
      p += st;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i < rows) *p = ElemOf<I>::down(x[i]);
    p += st;
  }
}

// ---------------------------------------------------------------- state
template <typename I, int DK, int DV>
struct StateMem {
  static constexpr int kPanels = DK / 64, kPanelS = DV * 128, kPlaneS = kPanels * kPanelS, kPlaneX = DV * 128;
  // Keys and queries: 64 rows of each to a panel, so that one operand of 128 rows has both.
  static constexpr int kPanelKQ = 2 * kTok, kPlaneKQ = kPanels * kPanelKQ, kStageKQ = kParts<I> * kPlaneKQ;
  static constexpr int S = 0, X = S + 2 * kPlaneS, W = X + 2 * kPlaneX, KQ = W + 2 * kPlaneX, T = KQ + 2 * kStageKQ, P = T + 2 * kTok,
                       kTiles = P + 2 * kTok;
};

enum StateBar { kGotKQ, kGotKQ2, kLoadedT, kLoadedP, kHalfSet, kStateSet, kRhsSet, kWritesSet, kReadDone, kSolveDone, kStateDone, kOutDone, kFactorsSet, kStateBars };

struct StateShared {
  uint64_t bar[kStateBars];
  uint32_t tmem;
  Factors f[2];
  float grown_q[3][kChunk];  // exp(G) rq: an output is written a chunk later than the factors are read
};

// One slice of a head's state, chunk after chunk. Tensor memory: S^T (128 x DK), twice K S and Q S, then E and
// after it P V', each in two halves.
template <typename I, int DK, int DV>
__global__ void __launch_bounds__(kThreads, 1) state_kernel(const DeltaFwd a) {
  using Mem = StateMem<I, DK, DV>;
  constexpr int P = kParts<I>;
  extern __shared__ __align__(1024) unsigned char mem[];
  StateShared& sh = *reinterpret_cast<StateShared*>(mem + Mem::kTiles);
  const DeltaDims& d = a.d;
  const int slices = d.slices, slice = blockIdx.x % slices, v0 = slice * DV, width = min(DV, d.dv - v0);
  const long long head = blockIdx.x / slices;
  const int b = (int)(head / d.H), h = (int)(head % d.H), hk = h / (d.H / d.Hk), chunks = d.chunks;
  const long long n0 = head * chunks, m0 = ((long long)b * d.Hk + hk) * chunks;
  const int tid = threadIdx.x, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < kStateBars; ++i)
      mbar_init(&sh.bar[i], i == kFactorsSet ? kChunk : i == kHalfSet || i == kStateSet || i == kRhsSet || i == kWritesSet ? kWorkers : 1);
    fence_barrier_init();
  }
  if (warp == kControl) tmem_alloc(&sh.tmem, 512);
  FactorParts parts;
  if (tid < kChunk && chunks > 0) {
    parts.read(a.keep, n0, m0, tid);
    parts.fill(sh.f[0], sh.grown_q[0], tid);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = sh.tmem;
  constexpr uint32_t cS = 0, cK = 128, cQ = 192, cE = 384, cP = cE;  // cK and cQ again 128 columns on; E is read before P V' comes
  Waiter wait{a.err};
  if (warp == kControl) {
    if ((tid & 31) == 0) {
      const auto load_kq = [&](int c) {
        uint64_t* bar = &sh.bar[c & 1 ? kGotKQ2 : kGotKQ];
        mbar_arrive_expect_tx(bar, Mem::kStageKQ);
        unsigned char* to = mem + Mem::KQ + (c & 1) * Mem::kStageKQ;
        const long long from = (m0 + c) * (Mem::kStageKQ / 2);
#pragma unroll
        for (int i = 0; i < P * Mem::kPanels; ++i) {
          bulk_load(to + i * Mem::kPanelKQ, a.keep.keys + from + i * kTok, kTok, bar);
          bulk_load(to + i * Mem::kPanelKQ + kTok, a.keep.queries + from + i * kTok, kTok, bar);
        }
      };
      const auto load_square = [&](int to, const unsigned char* from, int c, uint64_t* bar) {
        mbar_arrive_expect_tx(bar, 2 * kTok);
        bulk_load(mem + to, from + (n0 + c) * 2 * kTok, 2 * kTok, bar);
      };
      for (int c = 0; c < 2 && c < chunks; ++c) load_kq(c);
      if (chunks > 0) {
        load_square(Mem::T, a.keep.solve, 0, &sh.bar[kLoadedT]);
        load_square(Mem::P, a.keep.attend, 0, &sh.bar[kLoadedP]);
      }
      const uint32_t base = smem_u32(mem);
      const Operand S{base + Mem::S, Mem::kPanelS}, X{base + Mem::X, Mem::kPlaneX}, W{base + Mem::W, Mem::kPlaneX}, T{base + Mem::T, kTok},
          At{base + Mem::P, kTok};
      const auto store_state = [&](int c) {
        if (a.keep.states == nullptr) return;
        bulk_store(a.keep.states + ((head * chunks + c) * slices + slice) * 2 * Mem::kPlaneS, mem + Mem::S, 2 * Mem::kPlaneS);
        bulk_commit();
      };
      int c = 0;
      for (; c < chunks; ++c) {
        const Operand KQ{base + Mem::KQ + (c & 1) * Mem::kStageKQ, Mem::kPanelKQ};
        if (!wait(&sh.bar[c & 1 ? kGotKQ2 : kGotKQ], c >> 1)) break;
        if constexpr (Mem::kPanels == 2) {  // the first half's products run while the second half is set
          if (!wait(&sh.bar[kHalfSet], c)) break;
          tc_fence_after();
          multiply_parts<4, 128, false, false, 2, P>(tm + cK + (c & 1) * 128, S, Mem::kPlaneS, KQ, Mem::kPlaneKQ, false);
        }
        if (!wait(&sh.bar[kStateSet], c)) break;
        tc_fence_after();
        constexpr int kLast = Mem::kPanels - 1;
        multiply_parts<4, 128, false, false, 2, P>(tm + cK + (c & 1) * 128, Operand{S.addr + kLast * Mem::kPanelS, Mem::kPanelS}, Mem::kPlaneS,
                                                   Operand{KQ.addr + kLast * Mem::kPanelKQ, Mem::kPanelKQ}, Mem::kPlaneKQ, kLast > 0);
        tc_commit(&sh.bar[kReadDone]);
        store_state(c);
        if (!wait(&sh.bar[kRhsSet], c)) break;
        if (!wait(&sh.bar[kLoadedT], c)) break;
        tc_fence_after();
        multiply_wide<4, 128, false, false, 2>(tm + cE, X, Mem::kPlaneX, T, false);
        bulk_read_one_left();  // the last chunk's writes are copied: their place may be written once this product is done
        tc_commit(&sh.bar[kSolveDone]);
        if (!wait(&sh.bar[kWritesSet], c)) break;
        if (c + 1 < chunks) load_square(Mem::T, a.keep.solve, c + 1, &sh.bar[kLoadedT]);
        tc_fence_after();
        multiply_parts<4, DK, false, true, 2, P>(tm + cS, X, Mem::kPlaneX, KQ, Mem::kPlaneKQ, true);
        bulk_read_done();  // so is the state
        tc_commit(&sh.bar[kStateDone]);
        if (!wait(&sh.bar[kLoadedP], c)) break;
        multiply_wide<4, 128, false, false, 2>(tm + cP, W, Mem::kPlaneX, At, false);
        tc_commit(&sh.bar[kOutDone]);
        if (a.keep.writes != nullptr) {
          bulk_store(a.keep.writes + ((n0 + c) * slices + slice) * 2 * Mem::kPlaneX, mem + Mem::W, 2 * Mem::kPlaneX);
          bulk_commit();
        }
        if (!wait(&sh.bar[kStateDone], c)) break;
        if (c + 2 < chunks) load_kq(c + 2);
        if (!wait(&sh.bar[kOutDone], c)) break;
        if (c + 1 < chunks) load_square(Mem::P, a.keep.attend, c + 1, &sh.bar[kLoadedP]);
      }
      bulk_done();
    }
  } else if (warp > kControl) {
    const int i = tid - kWorkers - 32;
    for (int c = 0; c + 1 < chunks; ++c) {
      parts.read(a.keep, n0 + c + 1, m0 + c + 1, i);
      if (!wait(&sh.bar[kStateSet], c)) break;  // all are done with the factors before this chunk's
      parts.fill(sh.f[(c + 1) & 1], sh.grown_q[(c + 1) % 3], i);
      mbar_arrive(&sh.bar[kFactorsSet]);
    }
  } else {
    const Seat seat;
    const bool there = seat.row < DV, in = seat.row < width;  // a lane of the slice; one with an element of the head
    const int tt = seat.part * 16;
    const I* v = head_at<I>(a.v, b, 0, h) + v0 + seat.row;
    I* out = reinterpret_cast<I*>(a.out) + ((long long)b * d.T * d.H + h) * d.dv + v0 + seat.row;
    const long long step = (long long)d.H * d.dv;
    constexpr int kCols = DK / 4;  // of a worker's quarter of a state's row
    // Writes the state's row as halves into the tile, and scaled into tensor memory.
    const auto set_state = [&](const float (&f)[16], int col, float left) {
      if (there)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float x[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = f[p * 8 + k];
          unsigned char* to = mem + Mem::S + (col >> 6) * Mem::kPanelS + piece_at(seat.row, ((col >> 3) & 7) + p);
          put8(to, to + Mem::kPlaneS, x);
        }
      uint32_t r[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) r[k] = __float_as_uint(f[k] * left);
      tmem_st_32x32b_x16(tm + seat.lanes + cS + col, r);
    };
    const auto put_out = [&](int c) {  // the output of chunk c: Q S and P V' are done
      const uint32_t flip = (c & 1) * 128;
      float x[16], y[16];
      tmem_sum(tm + seat.lanes + cP + tt, tm + seat.lanes + cP + 64 + tt, y);
      tmem_row(tm + seat.lanes + cQ + flip + tt, x);
      if (!in) return;
      const float* by = sh.grown_q[c % 3] + tt;
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = fmaf(by[i], x[i], y[i]);
      const int t = c * kChunk + tt;
      put_column(out + t * step, step, d.T - t, y);
    };
    I x[16];
    const auto take_values = [&](int c) {
      if (in) column_of(v + (long long)(c * kChunk + tt) * a.v.st, a.v.st, d.T - c * kChunk - tt, x);
    };
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = ElemOf<I>::down(0.f);
    if (chunks > 0) take_values(0);
    for (int c = 0; c <= chunks; ++c) {
      if (c > 0 && (!wait(&sh.bar[kStateDone], c - 1) || (c < chunks && !wait(&sh.bar[kFactorsSet], c - 1)))) break;
      tc_fence_after();
      const Factors& fac = sh.f[c & 1];
      const float left = c < chunks ? fac.left : 0.f;
#pragma unroll
      for (int k = 0; k < kCols / 16; ++k) {
        const int col = k * 64 + seat.part * 16;
        float f[16];
        if (c > 0) {
          tmem_row(tm + seat.lanes + cS + col, f);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            f[i] = a.first != nullptr && in && col + i < d.dk ? a.first[(head * d.dk + col + i) * d.dv + v0 + seat.row] : 0.f;
        }
        if (c == chunks && a.last != nullptr && in) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (col + i < d.dk) a.last[(head * d.dk + col + i) * d.dv + v0 + seat.row] = f[i];
        }
        set_state(f, col, left);
        if (k + 1 < kCols / 16) hand_over(&sh.bar[kHalfSet]);
      }
      tmem_st_wait();
      hand_over(&sh.bar[kStateSet]);
      if (c > 0) {
        if (!wait(&sh.bar[kOutDone], c - 1)) break;
        tc_fence_after();
        put_out(c - 1);
      }
      if (c == chunks) break;
      if (!wait(&sh.bar[kReadDone], c)) break;
      tc_fence_after();
      float f[16];
      tmem_row(tm + seat.lanes + cK + (c & 1) * 128 + tt, f);
      if (there) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float y[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) y[k] = fmaf(-fac.grown_k[tt + p * 8 + k], f[p * 8 + k], ElemOf<I>::up(x[p * 8 + k]));
          unsigned char* to = mem + Mem::X + piece_at(seat.row, seat.part * 2 + p);
          put8(to, to + Mem::kPlaneX, y);
        }
      }
      hand_over(&sh.bar[kRhsSet]);
      if (c + 1 < chunks) take_values(c + 1);
      if (!wait(&sh.bar[kSolveDone], c)) break;
      tc_fence_after();
      tmem_sum(tm + seat.lanes + cE + tt, tm + seat.lanes + cE + 64 + tt, f);
      if (there) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float y[8];
          const int at = piece_at(seat.row, seat.part * 2 + p);
#pragma unroll
          for (int k = 0; k < 8; ++k) y[k] = fac.beta[tt + p * 8 + k] * f[p * 8 + k];
          put8(mem + Mem::W + at, mem + Mem::W + Mem::kPlaneX + at, y);
#pragma unroll
          for (int k = 0; k < 8; ++k) y[k] *= fac.left_k[tt + p * 8 + k];
          put8(mem + Mem::X + at, mem + Mem::X + Mem::kPlaneX + at, y);
        }
      }
      hand_over(&sh.bar[kWritesSet]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kControl) {
    tc_fence_after();
    tmem_dealloc(tm, 512);
  }
}

// ---------------------------------------------------------------- dstate
template <typename I, int DK, int DV>
struct DstateMem {
  static constexpr int kPanels = DK / 64, kParts_ = kParts<I>, kPanelS = DV * 128, kPlaneS = kPanels * kPanelS, kPlaneX = DV * 128,
                       kPlaneK = kPanels * kTok;
  static constexpr int kStages = kParts<I> == 1 ? 2 : 1;  // of the keys, which a chunk's first and last product read
  // Y: diag(exp G rq) dO, then dV; O: dO
  static constexpr int S = 0, X = S + 2 * kPlaneS, Y = X + 2 * kPlaneX, O = Y + 2 * kPlaneX, K = O + kParts_ * kPlaneX,
                       Q = K + kStages * kParts_ * kPlaneK, P = Q + kParts_ * kPlaneK, T = P + 2 * kTok, kTiles = T + 2 * kTok;
};

enum DstateBar { kGotK, kGotK2, kGotQ, kGotT, kHalfDset, kDstateSet, kOutsSet, kGradSet, kReadsSet, kMixDone, kOutsDone, kBackDone, kDstateDone, kTilesFree, kPartsSet, kDstateBars };

struct DstateShared {
  uint64_t bar[kDstateBars];
  uint32_t tmem;
  Factors f[2];
  float grown_q[2][kChunk];  // exp(G) rq
};

// One slice of the gradient of a head's state, from the last chunk to the first. Tensor memory: dS^T (128 x DK), K dS',
// P^T dO and dV in two halves each.
template <typename I, int DK, int DV>
__global__ void __launch_bounds__(kThreads, 1) dstate_kernel(const DeltaBwd a) {
  using Mem = DstateMem<I, DK, DV>;
  constexpr int P = kParts<I>, kStages = Mem::kStages;
  extern __shared__ __align__(1024) unsigned char mem[];
  DstateShared& sh = *reinterpret_cast<DstateShared*>(mem + Mem::kTiles);
  const DeltaDims& d = a.d;
  const int slices = d.slices, slice = blockIdx.x % slices, v0 = slice * DV, width = min(DV, d.dv - v0);
  const long long head = blockIdx.x / slices;
  const int b = (int)(head / d.H), h = (int)(head % d.H), hk = h / (d.H / d.Hk), chunks = d.chunks;
  const long long n0 = head * chunks, m0 = ((long long)b * d.Hk + hk) * chunks;
  const int tid = threadIdx.x, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < kDstateBars; ++i)
      mbar_init(&sh.bar[i], i == kPartsSet ? kChunk : i == kHalfDset || i == kDstateSet || i == kOutsSet || i == kGradSet || i == kReadsSet ? kWorkers : 1);
    fence_barrier_init();
  }
  if (warp == kControl) tmem_alloc(&sh.tmem, 512);
  FactorParts parts;
  if (tid < kChunk && chunks > 0) {
    parts.read(a.keep, n0 + chunks - 1, m0 + chunks - 1, tid);
    parts.fill(sh.f[0], sh.grown_q[0], tid);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = sh.tmem;
  constexpr uint32_t cS = 0, cK = 128, cO = 192, cV = 320;
  Waiter wait{a.err};
  if (warp == kControl) {
    if ((tid & 31) == 0 && chunks > 0) {
      const auto load_k = [&](int r) {  // round r: chunk chunks - 1 - r
        uint64_t* bar = &sh.bar[kStages == 2 && (r & 1) ? kGotK2 : kGotK];
        mbar_arrive_expect_tx(bar, P * Mem::kPlaneK);
        bulk_load(mem + Mem::K + r % kStages * P * Mem::kPlaneK, a.keep.keys + (m0 + chunks - 1 - r) * P * Mem::kPlaneK, P * Mem::kPlaneK, bar);
      };
      const auto load_q = [&](int r) {
        mbar_arrive_expect_tx(&sh.bar[kGotQ], P * Mem::kPlaneK + 2 * kTok);
        bulk_load(mem + Mem::Q, a.keep.queries + (m0 + chunks - 1 - r) * P * Mem::kPlaneK, P * Mem::kPlaneK, &sh.bar[kGotQ]);
        bulk_load(mem + Mem::P, a.keep.attend + (n0 + chunks - 1 - r) * 2 * kTok, 2 * kTok, &sh.bar[kGotQ]);
      };
      const auto load_t = [&](int r) {
        mbar_arrive_expect_tx(&sh.bar[kGotT], 2 * kTok);
        bulk_load(mem + Mem::T, a.keep.solve + (n0 + chunks - 1 - r) * 2 * kTok, 2 * kTok, &sh.bar[kGotT]);
      };
      for (int r = 0; r < kStages && r < chunks; ++r) load_k(r);
      load_q(0);
      load_t(0);
      const uint32_t base = smem_u32(mem);
      const Operand S{base + Mem::S, Mem::kPanelS}, X{base + Mem::X, Mem::kPlaneX}, Y{base + Mem::Y, Mem::kPlaneX},
          O{base + Mem::O, Mem::kPlaneX}, Q{base + Mem::Q, kTok}, At{base + Mem::P, kTok}, T{base + Mem::T, kTok};
      for (int r = 0; r < chunks; ++r) {
        const Operand K{base + Mem::K + r % kStages * P * Mem::kPlaneK, kTok};
        if (!wait(&sh.bar[kStages == 2 && (r & 1) ? kGotK2 : kGotK], kStages == 2 ? r >> 1 : r)) break;
        if constexpr (Mem::kPanels == 2) {
          if (!wait(&sh.bar[kHalfDset], r)) break;
          tc_fence_after();
          multiply_parts<4, 64, false, false, 2, P>(tm + cK, S, Mem::kPlaneS, K, Mem::kPlaneK, false);
        }
        if (!wait(&sh.bar[kDstateSet], r)) break;
        tc_fence_after();
        constexpr int kLast = Mem::kPanels - 1;
        multiply_parts<4, 64, false, false, 2, P>(tm + cK, Operand{S.addr + kLast * Mem::kPanelS, Mem::kPanelS}, Mem::kPlaneS,
                                                  Operand{K.addr + kLast * kTok, kTok}, Mem::kPlaneK, kLast > 0);
        if (!wait(&sh.bar[kOutsSet], r)) break;
        if (!wait(&sh.bar[kGotQ], r)) break;
        tc_fence_after();
        multiply_wide<4, 128, false, true, P>(tm + cO, O, Mem::kPlaneX, At, false);
        tc_commit(&sh.bar[kMixDone]);
        multiply_parts<4, DK, false, true, 2, P>(tm + cS, Y, Mem::kPlaneX, Q, Mem::kPlaneK, true);
        tc_commit(&sh.bar[kOutsDone]);
        const long long at_n = (n0 + chunks - 1 - r) * slices + slice;
        bulk_store(a.dstates + at_n * 2 * Mem::kPlaneS, mem + Mem::S, 2 * Mem::kPlaneS);
        bulk_store(a.douts + at_n * P * Mem::kPlaneX, mem + Mem::O, P * Mem::kPlaneX);
        bulk_commit();
        if (!wait(&sh.bar[kGradSet], r)) break;
        if (!wait(&sh.bar[kGotT], r)) break;
        tc_fence_after();
        multiply_wide<4, 128, false, true, 2>(tm + cV, X, Mem::kPlaneX, T, false);
        tc_commit(&sh.bar[kBackDone]);
        if (!wait(&sh.bar[kOutsDone], r)) break;
        if (r + 1 < chunks) load_q(r + 1);
        if (!wait(&sh.bar[kReadsSet], r)) break;
        if (r + 1 < chunks) load_t(r + 1);
        tc_fence_after();
        multiply_parts<4, DK, false, true, 2, P>(tm + cS, X, Mem::kPlaneX, K, Mem::kPlaneK, true);
        bulk_read_done();  // dS' and dO are copied: their places may be written once this product is done
        tc_commit(&sh.bar[kDstateDone]);
        bulk_store(a.dreads + at_n * 2 * Mem::kPlaneX, mem + Mem::Y, 2 * Mem::kPlaneX);
        bulk_commit();
        bulk_read_done();
        mbar_arrive(&sh.bar[kTilesFree]);
        if (!wait(&sh.bar[kDstateDone], r)) break;
        if (r + kStages < chunks) load_k(r + kStages);
      }
      bulk_done();
    }
  } else if (warp > kControl) {
    const int i = tid - kWorkers - 32;
    for (int r = 0; r + 1 < chunks; ++r) {
      parts.read(a.keep, n0 + chunks - 2 - r, m0 + chunks - 2 - r, i);
      if (!wait(&sh.bar[kDstateSet], r)) break;  // all are done with the factors before this chunk's
      parts.fill(sh.f[(r + 1) & 1], sh.grown_q[(r + 1) & 1], i);
      mbar_arrive(&sh.bar[kPartsSet]);
    }
  } else {
    const Seat seat;
    const bool there = seat.row < DV, in = seat.row < width;
    const int tt = seat.part * 16;
    const long long step = (long long)d.H * d.dv, at_head = ((long long)b * d.T * d.H + h) * d.dv + v0 + seat.row;
    const I* go = reinterpret_cast<const I*>(a.g_out) + at_head;
    I* dv = reinterpret_cast<I*>(a.dv) + at_head;
    constexpr int kCols = DK / 4;
    I x[16];
    const auto take_outs = [&](int c) {
      if (in) column_of(go + (c * kChunk + tt) * step, step, d.T - c * kChunk - tt, x);
    };
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = ElemOf<I>::down(0.f);
    if (chunks > 0) take_outs(chunks - 1);
    for (int r = 0; r <= chunks; ++r) {
      const int c = chunks - 1 - r;
      if (r > 0 && (!wait(&sh.bar[kDstateDone], r - 1) || (c >= 0 && !wait(&sh.bar[kPartsSet], r - 1)))) break;
      tc_fence_after();
      const Factors& fac = sh.f[r & 1];
      const float left = c >= 0 ? fac.left : 0.f;
#pragma unroll
      for (int k = 0; k < kCols / 16; ++k) {
        const int col = k * 64 + seat.part * 16;
        float f[16];
        if (r > 0) {
          tmem_row(tm + seat.lanes + cS + col, f);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            f[i] = a.g_last != nullptr && in && col + i < d.dk ? a.g_last[(head * d.dk + col + i) * d.dv + v0 + seat.row] : 0.f;
        }
        if (c < 0) {
          if (a.dfirst != nullptr && in) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (col + i < d.dk) a.dfirst[(head * d.dk + col + i) * d.dv + v0 + seat.row] = f[i];
          }
          continue;
        }
        if (there) {
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = f[p * 8 + i];
            unsigned char* to = mem + Mem::S + (col >> 6) * Mem::kPanelS + piece_at(seat.row, ((col >> 3) & 7) + p);
            put8(to, to + Mem::kPlaneS, y);
          }
        }
        uint32_t u[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(f[i] * left);
        tmem_st_32x32b_x16(tm + seat.lanes + cS + col, u);
        if (k + 1 < kCols / 16) hand_over(&sh.bar[kHalfDset]);
      }
      if (c < 0) break;
      tmem_st_wait();
      hand_over(&sh.bar[kDstateSet]);
      if (r > 0 && !wait(&sh.bar[kTilesFree], r - 1)) break;  // dV is copied
      if (there) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float y[8];
          const int at = piece_at(seat.row, seat.part * 2 + p);
#pragma unroll
          for (int k = 0; k < 8; ++k) y[k] = ElemOf<I>::up(x[p * 8 + k]);
          if constexpr (P == 2) put8(mem + Mem::O + at, mem + Mem::O + Mem::kPlaneX + at, y);
          else *reinterpret_cast<uint4*>(mem + Mem::O + at) = raw_down<I, uint4>(y);
#pragma unroll
          for (int k = 0; k < 8; ++k) y[k] *= sh.grown_q[r & 1][tt + p * 8 + k];
          put8(mem + Mem::Y + at, mem + Mem::Y + Mem::kPlaneX + at, y);
        }
      }
      hand_over(&sh.bar[kOutsSet]);
      if (c > 0) take_outs(c - 1);
      if (!wait(&sh.bar[kMixDone], r)) break;
      tc_fence_after();
      float f[16], y16[16];
      tmem_sum(tm + seat.lanes + cO + tt, tm + seat.lanes + cO + 64 + tt, y16);
      tmem_row(tm + seat.lanes + cK + tt, f);
      if (there) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float y[8];
          const int at = piece_at(seat.row, seat.part * 2 + p);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int i = p * 8 + k;
            y[k] = fac.beta[tt + i] * fmaf(fac.left_k[tt + i], f[i], y16[i]);
          }
          put8(mem + Mem::X + at, mem + Mem::X + Mem::kPlaneX + at, y);
        }
      }
      hand_over(&sh.bar[kGradSet]);
      if (!wait(&sh.bar[kBackDone], r) || !wait(&sh.bar[kOutsDone], r)) break;  // the solve, and Y read
      tc_fence_after();
      tmem_sum(tm + seat.lanes + cV + tt, tm + seat.lanes + cV + 64 + tt, f);
      if (there) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float y[8];
          const int at = piece_at(seat.row, seat.part * 2 + p);
#pragma unroll
          for (int k = 0; k < 8; ++k) y[k] = f[p * 8 + k];
          put8(mem + Mem::Y + at, mem + Mem::Y + Mem::kPlaneX + at, y);
#pragma unroll
          for (int k = 0; k < 8; ++k) y[k] *= -fac.grown_k[tt + p * 8 + k];
          put8(mem + Mem::X + at, mem + Mem::X + Mem::kPlaneX + at, y);
        }
      }
      hand_over(&sh.bar[kReadsSet]);
      const int t = c * kChunk + tt;
      if (in) put_column(dv + t * step, step, d.T - t, f);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kControl) {
    tc_fence_after();
    tmem_dealloc(tm, 512);
  }
}

template <typename I, int DK, int DV>
void state(const DeltaFwd& a, cudaStream_t s) {
  constexpr int bytes = StateMem<I, DK, DV>::kTiles + (int)sizeof(StateShared);
  static_assert(bytes <= 227 * 1024, "shared memory");
  cudaFuncSetAttribute(state_kernel<I, DK, DV>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  state_kernel<I, DK, DV><<<(unsigned)(a.d.B * a.d.H * a.d.slices), kThreads, bytes, s>>>(a);
}

template <typename I, int DK, int DV>
void dstate(const DeltaBwd& a, cudaStream_t s) {
  constexpr int bytes = DstateMem<I, DK, DV>::kTiles + (int)sizeof(DstateShared);
  static_assert(bytes <= 227 * 1024, "shared memory");
  cudaFuncSetAttribute(dstate_kernel<I, DK, DV>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  dstate_kernel<I, DK, DV><<<(unsigned)(a.d.B * a.d.H * a.d.slices), kThreads, bytes, s>>>(a);
}

template <typename I>
void state_of(const DeltaFwd& a, cudaStream_t s) {
  if (a.d.slice == 64) return a.d.dk <= 64 ? state<I, 64, 64>(a, s) : state<I, 128, 64>(a, s);
  if constexpr (kParts<I> == 1)
    if (a.d.dk > 64) return state<I, 128, 128>(a, s);
  state<I, 64, 128>(a, s);
}

template <typename I>
void dstate_of(const DeltaBwd& a, cudaStream_t s) {
  if (a.d.slice == 64) return a.d.dk <= 64 ? dstate<I, 64, 64>(a, s) : dstate<I, 128, 64>(a, s);
  if constexpr (kParts<I> == 1)
    if (a.d.dk > 64) return dstate<I, 128, 128>(a, s);
  dstate<I, 64, 128>(a, s);
}

}  // namespace

void delta_state(const DeltaFwd& a, cudaStream_t s) {
  a.d.type == Elem::kBF16 ? state_of<bf16>(a, s) : state_of<__half>(a, s);
}

void delta_dstate(const DeltaBwd& a, cudaStream_t s) {
  a.d.type == Elem::kBF16 ? dstate_of<bf16>(a, s) : dstate_of<__half>(a, s);
}

}  // namespace bw
