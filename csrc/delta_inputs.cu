// Gated delta rule in chunks, backward: the gradients of q, k and the gates (formulas in delta_state.cu).
//
// A CTA to each chunk of a value head; the value heads of one key head are a cluster, whose CTAs add their rows of dq and dk
// over distributed shared memory in the order of the heads. Products, all with 128 lanes of tensor memory:
//     S [dO | dV]^T, dS' V'^T  lanes are the elements of a key row, columns the tokens
//     [dO | dV] V'^T           dP in lanes 0..63, dL in 64..127: both gradients side by side as the rows of one operand
//     [q | k] k^T              beside them, for what passes the gates
//     K^T W, K^T W', Q^T W     W = dP D rq_i rk_j and dL D rk_i rk_j: q and k go in as given, their lengths in the small matrix
// so that all scalings of tokens are by columns, in fp32, when the sums leave tensor memory. S comes first: q, k and the small
// matrices take its place where heads are large.
//
// What bounds it: one CTA of 208 KB of tiles to an SM, whose steps (tiles in, three products, the small matrices, three more, rows
// out) wait for one another: 2,600 instructions a warp fill 39 % of the issue slots, memory runs at a quarter of its rate. 4 x
// 2048 tokens, 16 key and 32 value heads of 128 x 128, bf16: 395 us (1734 on instructions of single warps); 1.05 GB to read
// and write, 160 us. Clusters that stay and take chunk after chunk: 451 us, the last rows and the next tiles share their place.
#include <cooperative_groups.h>

#include "delta_tiles.cuh"

namespace bw {
namespace {

namespace cg = cooperative_groups;

template <typename I, int DK, int DV>
struct InputsMem {
  static constexpr int kPanels = DK / 64, kPanelS = DV * 128, kPlaneS = kPanels * kPanelS, kPlaneX = DV * 128;
  // dS'; V'; the stack: dO and dV, the high halves before the low ones (dO in bf16 has none); S; q and k; the small matrices.
  // The largest state takes all there is: q, k and the small matrices then come where S was. In the end, from the start on: all
  // heads' parts of the owned rows, a multiple of 16 (at most 32 from each of seven heads).
  static constexpr int ldF = DK + 4, kRows = 7 * 32 * ldF * 4;
  static constexpr int kKeys = 2 * kParts<I> * kPanels * kTok, kSquares = 4 * kTok;
  static constexpr int D = 0, V = D + 2 * kPlaneS, O = V + 2 * kPlaneX, G = O + kPlaneX, Ol = G + kPlaneX,
                       Gl = Ol + (kParts<I> == 2 ? kPlaneX : 0), S = Gl + kPlaneX, kUsed = S + 2 * kPlaneS,
                       kEnd = kUsed > kRows ? kUsed : align1k(kRows);
  // Panels of q and of k take turns, so that their rows are one operand's 128; parts are kPart apart.
  static constexpr int kPanelK = 2 * kTok, kPart = kPanels * kPanelK;
  static constexpr bool kShared = kEnd + kKeys + kSquares > 220 * 1024;
  static constexpr bool kAllShared = kShared && kKeys + kSquares <= 2 * kPlaneS;
  static constexpr int Q = kShared ? S : kEnd, K = Q + kTok, W = kShared && !kAllShared ? kEnd : Q + kKeys, N = W + 2 * kTok,
                       kTiles = kAllShared ? kEnd : N + 2 * kTok;
  static_assert(!kShared || kKeys <= 2 * kPlaneS, "room where S was");
  static_assert(kRows <= Q, "the rows of q and k stay");
  static constexpr int kBytes = kTiles;
};

enum InputsBar { kGotQK, kGotV, kGotS, kGotD, kMixDone, kReadS, kReadD, kMixSet, kGramDone, kGramRead, kAllDone, kTaken, kInputsBars };

struct InputsShared {
  uint64_t bar[kInputsBars];
  uint32_t tmem;
  float2 G[kChunk];
  float rk[kChunk], rq[kChunk], beta[kChunk];
  float4 by[kChunk];                // what a token's sums are multiplied by: its query's read, its key's read and its write
  float kept;                       // exp(G_63)
  float2 gate[kChunk];              // log-decay, and its derivative by a
  float written[kChunk];            // V' . dV
  float read[4][kChunk];            // what S gives to a token, of each quarter of a key head
  float left_over[4][kChunk];       // what a token gives to S'
  float near[4][kChunk];            // what the tokens of t's sixteen before t give to t and those behind it: of half of P, of L each
  float far[kChunk / 16][2 * kChunk];  // what each sixteen tokens give to a later one: P, L
  float handed[kControl];           // S to S'

};

// Adds to the sums of lane (i, i / 2 % 4) the products of bf16 pairs that lie in the same places of two matrices, each in halves:
// a 16 x 8 product of which only the diagonals are wanted, a lane's words with the same lane's, takes a sixth of the
// instructions that unpack and multiply them.
__device__ __forceinline__ void dot_halves(float (&c)[4], uint32_t h0, uint32_t l0, uint32_t h1, uint32_t l1, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(h0), "r"(l0), "r"(h1), "r"(l1), "r"(b0), "r"(b1));
}

// Stores to the shared memory of a CTA of the cluster.
__device__ __forceinline__ uint32_t rank_addr(uint32_t at, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
  return r;
}
__device__ __forceinline__ void store_at(uint32_t at, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}

// Adds 32 values of each of 32 lanes over the lanes: lane l ends with the sum of value l.
__device__ __forceinline__ float lanes_fold(float (&x)[32]) {
#pragma unroll
  for (int n = 16; n > 0; n >>= 1) {
    const bool up = threadIdx.x & n;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float send = up ? x[i] : x[i + n], keep = up ? x[i + n] : x[i];
      x[i] = keep + __shfl_xor_sync(0xffffffffu, send, n);
    }
  }
  return x[0];
}

// Adds 16 values of each of 32 lanes over the lanes: lane l ends with the sum of value l % 16.
__device__ __forceinline__ float lanes_fold16(float (&x)[16]) {
#pragma unroll
  for (int n = 8; n > 0; n >>= 1) {
    const bool up = threadIdx.x & n;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float send = up ? x[i] : x[i + n], keep = up ? x[i + n] : x[i];
      x[i] = keep + __shfl_xor_sync(0xffffffffu, send, n);
    }
  }
  return x[0] + __shfl_xor_sync(0xffffffffu, x[0], 16);
}

template <typename I, int DK, int DV>
__global__ void __launch_bounds__(kWorkers + 32, 1) inputs_kernel(const DeltaBwd a) {
  using Mem = InputsMem<I, DK, DV>;
  constexpr int P = kParts<I>, kVs = DV / 16;
  extern __shared__ __align__(1024) unsigned char mem[];
  InputsShared& sh = *reinterpret_cast<InputsShared*>(mem + Mem::kBytes);
  const DeltaDims& d = a.d;
  const int group = d.H / d.Hk, chunks = d.chunks, slices = d.slices;
  // blockIdx.x = (batch * Hk + key head, chunk, head within the group): the last runs over the cluster
  const int hg = blockIdx.x % group;
  const long long rest = blockIdx.x / group, bk = rest / chunks;
  const int c = (int)(rest % chunks), b = (int)(bk / d.Hk), hk = (int)(bk % d.Hk), h = hk * group + hg;
  const long long head = (long long)b * d.H + h, n = head * chunks + c, m = bk * chunks + c;
  const int t0 = c * kChunk, rows = min(kChunk, d.T - t0);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const auto state_at = [&](int chunk, int s) { return a.keep.states + ((head * chunks + chunk) * slices + s) * 2 * Mem::kPlaneS; };
  const auto load_slice = [&](int s) {
    const long long at = n * slices + s;
    mbar_arrive_expect_tx(&sh.bar[kGotV], (4 + P) * Mem::kPlaneX);
    bulk_load(mem + Mem::V, a.keep.writes + at * 2 * Mem::kPlaneX, 2 * Mem::kPlaneX, &sh.bar[kGotV]);
    bulk_load(mem + Mem::O, a.douts + at * P * Mem::kPlaneX, Mem::kPlaneX, &sh.bar[kGotV]);
    if (P == 2) bulk_load(mem + Mem::Ol, a.douts + (at * P + 1) * Mem::kPlaneX, Mem::kPlaneX, &sh.bar[kGotV]);
    bulk_load(mem + Mem::G, a.dreads + at * 2 * Mem::kPlaneX, Mem::kPlaneX, &sh.bar[kGotV]);
    bulk_load(mem + Mem::Gl, a.dreads + at * 2 * Mem::kPlaneX + Mem::kPlaneX, Mem::kPlaneX, &sh.bar[kGotV]);
    mbar_arrive_expect_tx(&sh.bar[kGotS], 2 * Mem::kPlaneS);
    bulk_load(mem + Mem::S, state_at(c, s), 2 * Mem::kPlaneS, &sh.bar[kGotS]);
    mbar_arrive_expect_tx(&sh.bar[kGotD], 2 * Mem::kPlaneS);
    bulk_load(mem + Mem::D, a.dstates + at * 2 * Mem::kPlaneS, 2 * Mem::kPlaneS, &sh.bar[kGotD]);
  };
  const auto load_keys = [&] {
    mbar_arrive_expect_tx(&sh.bar[kGotQK], 2 * P * Mem::kPanels * kTok);
#pragma unroll
    for (int i = 0; i < P * Mem::kPanels; ++i) {
      bulk_load(mem + Mem::Q + i * Mem::kPanelK, a.keep.queries + m * P * Mem::kPanels * kTok + i * kTok, kTok, &sh.bar[kGotQK]);
      bulk_load(mem + Mem::K + i * Mem::kPanelK, a.keep.keys + m * P * Mem::kPanels * kTok + i * kTok, kTok, &sh.bar[kGotQK]);
    }
  };
  if (tid == kWorkers) {
    for (int i = 0; i < kInputsBars; ++i) mbar_init(&sh.bar[i], i == kMixSet || i == kGramRead || i == kTaken ? kWorkers : 1);
    fence_barrier_init();
    fence_proxy_async_smem();
    load_slice(0);
    if (Mem::kShared) {
      bulk_prefetch(a.keep.queries + m * P * Mem::kPanels * kTok, P * Mem::kPanels * kTok);
      bulk_prefetch(a.keep.keys + m * P * Mem::kPanels * kTok, P * Mem::kPanels * kTok);
    } else {
      load_keys();
    }
  }
  __syncwarp();
  if (warp == kControl) tmem_alloc(&sh.tmem, 512);
  if (tid < kChunk) {
    const float2 G = a.keep.total[n * kChunk + tid], end = a.keep.total[n * kChunk + kChunk - 1];
    sh.G[tid] = G;
    sh.rk[tid] = a.keep.rk[m * kChunk + tid];
    sh.rq[tid] = a.keep.rq[m * kChunk + tid];
    sh.beta[tid] = a.keep.beta[n * kChunk + tid];
    const float grown = __expf(G.x + G.y);
    sh.by[tid] = make_float4(sh.rq[tid] * grown, -sh.rk[tid] * grown, sh.rk[tid] * decay_between(end, G), 0.f);
    if (tid == kChunk - 1) sh.kept = grown;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = sh.tmem;
  const Seat seat;
  // The last two come when the small matrices' products, in the same place, are read.
  constexpr uint32_t cS = 0, cD = 128, cMix = 256, cLow = 384, cGram = 448, cQ = 256, cK = 384;
  Waiter wait{a.err};
  if (warp == kControl) {
    if (lane == 0) {
      const uint32_t base = smem_u32(mem);
      // The stack of high halves, and that of low ones; without a low half of dO the first 64 lanes of its product are not used.
      const Operand high{base + Mem::O, Mem::G - Mem::O}, low{base + (P == 2 ? Mem::Ol : Mem::O), Mem::Gl - (P == 2 ? Mem::Ol : Mem::O)},
          low_g{base + Mem::Gl, Mem::kPlaneX}, V{base + Mem::V, Mem::kPlaneX},
          S{base + Mem::S, Mem::kPanelS}, Sl{base + Mem::S + Mem::kPlaneS, Mem::kPanelS}, D{base + Mem::D, Mem::kPanelS},
          Dl{base + Mem::D + Mem::kPlaneS, Mem::kPanelS};
      for (int s = 0; s < slices; ++s) {
        const bool more = s > 0;
        if (!wait(&sh.bar[kGotV], s)) break;
        if (!wait(&sh.bar[kGotS], s)) break;
        multiply<kVs, 128, true, true>(tm + cS, S, high, more);
        multiply<kVs, 128, true, true>(tm + cS, Sl, high, true);
        if (P == 2) multiply<kVs, 128, true, true>(tm + cS, S, low, true);
        else multiply<kVs, 64, true, true>(tm + cS + 64, S, low_g, true);
        tc_commit(&sh.bar[kReadS]);
        multiply<kVs, 128, true, true>(tm + cMix, high, V, more);  // both halves of V' side by side
        multiply<kVs, 64, true, true>(P == 2 ? tm + cMix : tm + cLow, low, V, P == 2 || more);
        if (s == slices - 1) tc_commit(&sh.bar[kMixDone]);
        if (Mem::kShared && s == slices - 1) {
          if (!wait(&sh.bar[kReadS], s)) break;
          load_keys();
        }
        if (!wait(&sh.bar[kGotD], s)) break;
        multiply<kVs, 128, true, true>(tm + cD, D, V, more);
        multiply<kVs, 64, true, true>(tm + cD, Dl, V, true);
        if (s + 1 < slices) {  // the places are free once they are read, by the products and by the workers
          tc_commit(&sh.bar[kReadD]);
          if (!wait(&sh.bar[kReadS], s) || !wait(&sh.bar[kReadD], s) || !wait(&sh.bar[kTaken], s)) break;
          load_slice(s + 1);
        }
      }
      const Operand Q{base + Mem::Q, Mem::kPanelK}, K{base + Mem::K, Mem::kPanelK}, W{base + Mem::W, kTok}, N{base + Mem::N, kTok};
      if (wait(&sh.bar[kGotQK], 0)) {
        multiply_parts<DK / 16, 64, false, false, P, P>(tm + cGram, Q, Mem::kPart, K, Mem::kPart, false);  // [q | k] k^T
        tc_commit(&sh.bar[kGramDone]);
        if (wait(&sh.bar[kMixSet], 0)) {
          tc_fence_after();
          multiply_wide<4, 128, true, false, P>(tm + cQ, K, Mem::kPart, W, false);
          if (wait(&sh.bar[kGramRead], 0)) {
            tc_fence_after();
            multiply_wide<4, 128, true, true, P>(tm + cK, Q, Mem::kPart, W, false);
            multiply_wide<4, 128, true, false, P>(tm + cK, K, Mem::kPart, N, true);
            multiply_wide<4, 128, true, true, P>(tm + cK, K, Mem::kPart, N, true);
            tc_commit(&sh.bar[kAllDone]);
            wait(&sh.bar[kAllDone], 0);
          }
        }
      }
    }
  } else {
    float handed[4] = {0.f, 0.f, 0.f, 0.f};
    const int tt = seat.part * 16;  // its tokens
    float mix[16];
    // While the first tiles are on their way. Left to the warp that sums the gates' gradients, this held the CTA back (433 us, 391 with it here).
    if (tid < rows) {
      const Gate gate = gate_of(ElemOf<I>::up(*head_at<I>(a.g.a, b, t0 + tid, h)), load_any(a.g.a_log, a.g.a_log_type, h),
                                load_any(a.g.dt_bias, a.g.dt_bias_type, h));
      sh.gate[tid] = make_float2(gate.log_decay, -gate.rate * gate.slope);
    }
    for (int s = 0; s < slices; ++s) {
      const bool in = seat.row < min(DV, d.dv - s * DV);
      // The small matrices first, for the products that wait for them: row i of dP in lane i, of dL in lane 64 + i.
      if (s == slices - 1) {
        if (!wait(&sh.bar[kMixDone], 0)) break;
        tc_fence_after();
        const int i = seat.row & 63, j0 = seat.part * 16;
        const bool of_l = seat.row >= 64;
        float f[16];
        tmem_sum(tm + seat.lanes + cMix + j0, tm + seat.lanes + cMix + 64 + j0, f);
        if (P == 1) {
          float g[16];
          tmem_row(tm + seat.lanes + cLow + j0, g);
          if (of_l)
#pragma unroll
            for (int k = 0; k < 16; ++k) f[k] += g[k];
        }
        const float by = of_l ? -sh.rk[i] : sh.rq[i];
        const float2 Gi = sh.G[i];
        const int last = of_l ? i : i + 1;
        unsigned char* to = mem + (of_l ? Mem::N : Mem::W);
        if (Mem::kAllShared && !wait(&sh.bar[kReadS], s)) break;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float x[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int j = j0 + p * 8 + k;
            const float w = f[p * 8 + k] * by * (decay_between(Gi, sh.G[j]) * sh.rk[j]);
            mix[p * 8 + k] = x[k] = j < last ? w : 0.f;
            if (of_l && j == i) sh.written[i] = f[p * 8 + k];
          }
          const int at = piece_at(i, seat.part * 2 + p);
          put8(to + at, to + kTok + at, x);
        }
        hand_over(&sh.bar[kMixSet]);
      }
      // <dS', S>: both tiles have their elements at the same places. S may be gone from shared memory by then, but not from L2.
      const uint4* before = reinterpret_cast<const uint4*>(state_at(c, s));
      constexpr int kPieces = Mem::kPlaneS / 16, kMine = kPieces / kWorkers;
      static_assert(kPieces % kWorkers == 0, "whole rounds");
      uint4 ah[kMine], al[kMine];
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        ah[i] = __ldcs(before + i * kWorkers + tid);
        al[i] = __ldcs(before + kPieces + i * kWorkers + tid);
      }
      // What passes the gate of token t within the chunk: from the tokens of its sixteen before t here, from earlier sixteens by
      // the sums of their columns.
      if (s == slices - 1) {
        float x[16];
        if (!wait(&sh.bar[kGramDone], 0)) break;
        tc_fence_after();
        tmem_row(tm + seat.lanes + cGram + tt, x);
        tc_fence_before();
        mbar_arrive(&sh.bar[kGramRead]);
        float run = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float next = fmaf(mix[k], x[k], run);
          x[k] = (seat.row & 63) >= tt + k ? run : 0.f;
          run = next;
        }
        sh.far[seat.part][seat.row] = run;
        const float near = lanes_fold16(x);
        if (lane < 16) sh.near[warp & 3][tt + lane] = near;
      }
      if (!wait(&sh.bar[kGotD], s)) break;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const unsigned char* at = mem + Mem::D + (i * kWorkers + tid) * 16;
        const uint4 dh = *reinterpret_cast<const uint4*>(at), dl = *reinterpret_cast<const uint4*>(at + Mem::kPlaneS);
        dot_halves(handed, dh.x, dl.x, dh.y, dl.y, ah[i].x, ah[i].y);
        dot_halves(handed, dh.x, dl.x, dh.y, dl.y, al[i].x, al[i].y);
        dot_halves(handed, dh.z, dl.z, dh.w, dl.w, ah[i].z, ah[i].w);
        dot_halves(handed, dh.z, dl.z, dh.w, dl.w, al[i].z, al[i].w);
      }
      mbar_arrive(&sh.bar[kTaken]);
    }
    // The diagonals of rows 0..7 and 8..15: row r, column 2 (lane % 4) + j of lane 4 r + lane % 4.
    const int r = lane >> 2;
    const float mine = lanes_sum((lane & 3) != r >> 1 ? 0.f : r & 1 ? handed[1] + handed[3] : handed[0] + handed[2]);
    if (lane == 0) sh.handed[warp] = mine;
    wait(&sh.bar[kAllDone], 0);
  }
  // dq and dk of this head: r dq^ and r dk^ of the scaled rows. The CTAs of the cluster own a part of the rows of both each and
  // get them from all heads, where dS' and V' lay.
  cg::cluster_group cluster = cg::this_cluster();
  __syncwarp();
  if (group > 1) cluster.barrier_arrive();  // this one is done with its products
  float* F = reinterpret_cast<float*>(mem);
  const int own = (2 * kChunk / 16 + group - 1) / group * 16;  // rows of an owner: one for the 16 tokens of a worker
  float y[16], z[16];
  if (warp < kControl) {
    tc_fence_after();
    const int tt = seat.part * 16;
    float x[32], g[16];
    tmem_sum(tm + seat.lanes + cD + tt, tm + seat.lanes + cD + 64 + tt, z);
    tmem_rows(tm + seat.lanes + cS + tt, y, tm + seat.lanes + cS + 64 + tt, g);
    // What S gives to a token and what a token gives to S': over the lanes here, over the warps of a column later. The rows of q
    // and k still lie as tiles.
    const auto element = [&](int tile, int i) {
      const unsigned char* at = mem + tile + element_at(i, seat.row, Mem::kPanelK);
      float v = __bfloat162float(*reinterpret_cast<const bf16*>(at));
      if (P == 2) v += __bfloat162float(*reinterpret_cast<const bf16*>(at + Mem::kPart));
      return v;
    };
    const bool in = seat.row < DK;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float key = in ? element(Mem::K, tt + k) : 0.f, query = in ? element(Mem::Q, tt + k) : 0.f;
      const float4 by = sh.by[tt + k];
      const float gives = by.z * z[k], reads = by.y * g[k];
      y[k] *= by.x;
      x[k] = in ? fmaf(query, y[k], key * reads) : 0.f;
      x[16 + k] = in ? key * gives : 0.f;
      z[k] = reads + gives;
    }
    const float sum = lanes_fold(x);
    (lane < 16 ? sh.read : sh.left_over)[warp & 3][tt + (lane & 15)] = sum;
    tmem_sum(tm + seat.lanes + cQ + tt, tm + seat.lanes + cQ + 64 + tt, g);
#pragma unroll
    for (int k = 0; k < 16; ++k) y[k] += g[k];
    tmem_sum(tm + seat.lanes + cK + tt, tm + seat.lanes + cK + 64 + tt, g);
#pragma unroll
    for (int k = 0; k < 16; ++k) z[k] += g[k];
    tc_fence_before();
  }
  if (group > 1) cluster.barrier_wait();
  else __syncthreads();
  if (warp < kControl && seat.row < DK) {
    const auto put = [&](int r0, const float (&v)[16]) {
      const int owner = r0 / own;
      float* f = F + (hg * own + r0 % own) * Mem::ldF + seat.row;
      if (owner == hg) {
#pragma unroll
        for (int k = 0; k < 16; ++k) f[k * Mem::ldF] = v[k];
      } else {
        const uint32_t at = rank_addr(smem_u32(f), owner);
#pragma unroll
        for (int k = 0; k < 16; ++k) store_at(at + k * Mem::ldF * 4, v[k]);
      }
    };
    put(seat.part * 16, y);
    put(kChunk + seat.part * 16, z);
  }
  __syncwarp();
  if (group > 1) cluster.sync();
  else __syncthreads();
  if (warp == kControl) {
    tc_fence_after();
    tmem_dealloc(tm, 512);
    // The gates, two tokens a lane: from S to tokens from t on, from tokens of earlier sixteens, of t's own, before t to those from
    // t on, from tokens before t to S', and from S to S'. Rolled up: one warp waits for its instructions far longer than for these sums.
    const float handed = lanes_sum(lane < kControl ? sh.handed[lane] : 0.f);
    float dg[2] = {sh.kept * handed, sh.kept * handed}, far[2] = {0.f, 0.f};
#pragma unroll 1
    for (int q = 0; q <= kChunk / 16; ++q) {
      const bool reads = q == 0, gives = q == kChunk / 16;
      const int step = gives ? -1 : 1;
      float x[2] = {0.f, 0.f};
      for (int k = 0; k < 2; ++k) {
        const int i = 2 * lane + k;
        if (reads || gives) {
          for (int w = 0; w < 4; ++w) x[k] += reads ? sh.read[w][i] : sh.left_over[w][i];
        } else {
          x[k] = far[k] += sh.far[q - 1][i] + sh.far[q - 1][kChunk + i];
        }
      }
      float sum = x[0] + x[1];
#pragma unroll 1
      for (int o = 1; o < 32; o <<= 1) {
        const int from = lane + step * o;
        const float more = __shfl_sync(0xffffffffu, sum, from & 31);
        if ((from & 31) == from) sum += more;
      }
      const float next = __shfl_sync(0xffffffffu, sum, (lane + step) & 31);
      const float rest = lane == (gives ? 0 : 31) ? 0.f : next;
      if (reads || gives || lane / 8 == q) {
        dg[0] += gives ? rest : rest + x[1] + x[0];
        dg[1] += gives ? rest + x[0] : rest + x[1];
      }
    }
    float sum_log = 0.f, sum_bias = 0.f;
    for (int k = 0; k < 2; ++k) {
      const int i = 2 * lane + k;
      if (i >= rows) continue;
      for (int w = 0; w < 4; ++w) dg[k] += sh.near[w][i];
      const float da = dg[k] * sh.gate[i].y;
      const float beta = sh.beta[i];
      const float db = beta > 1e-20f ? (1.f - beta) * (sh.written[i] / beta) : 0.f;  // V' = beta E; below, db is under 1e-20 dV . E
      const long long to = ((long long)b * d.T + t0 + i) * d.H + h;
      reinterpret_cast<I*>(a.da)[to] = ElemOf<I>::down(da);
      reinterpret_cast<I*>(a.db)[to] = ElemOf<I>::down(db);
      sum_log = fmaf(dg[k], sh.gate[i].x, sum_log);
      sum_bias += da;
    }
    sum_log = lanes_sum(sum_log);
    sum_bias = lanes_sum(sum_bias);
    if (lane == 0) {
      a.part[n * 2] = sum_log;
      a.part[n * 2 + 1] = sum_bias;
    }
    return;
  }
  // The owned rows' sums over the heads in their order, a row's elements side by side in a warp, then back through the rows'
  // scaling: with x a row, r its reciprocal length and y the sum, dx = y - x r^2 (x . y). Four rows at a time.
  constexpr int kE = DK / 32;  // elements of a lane
  const auto row_of = [&](int tile, int i, float (&x)[kE]) {
    const unsigned char* at = mem + tile + element_at(i, lane * kE, Mem::kPanelK);
    float lo[kE];
    if constexpr (kE == 4) {
      raw_up<bf16>(*reinterpret_cast<const uint2*>(at), x);
      if (P == 2) raw_up<bf16>(*reinterpret_cast<const uint2*>(at + Mem::kPart), lo);
    } else {
      raw_up<bf16>(*reinterpret_cast<const uint32_t*>(at), x);
      if (P == 2) raw_up<bf16>(*reinterpret_cast<const uint32_t*>(at + Mem::kPart), lo);
    }
    if (P == 2)
#pragma unroll
      for (int k = 0; k < kE; ++k) x[k] += lo[k];
  };
  const long long width = (long long)d.Hk * d.dk, start = ((long long)b * d.T + t0) * width + (long long)hk * d.dk + lane * kE;
  const float shorter = 1.f / d.scale;
  const bool in = lane * kE < d.dk;
  for (int p0 = warp; p0 < own && hg * own + p0 < 2 * kChunk; p0 += 4 * kControl) {
    float y[4][kE], x[4][kE], dot[4];
    // The rows of a warp are 16 apart, an owner's a multiple of 16: all or none of each sixteen. Rows behind the last are read as the first.
    const int most = min(own, 2 * kChunk - hg * own);
    int place[4];
#pragma unroll
    for (int n4 = 0; n4 < 4; ++n4) {
      place[n4] = p0 + n4 * kControl < most ? p0 + n4 * kControl : p0;
      const int r = hg * own + place[n4];
      row_of(r >= kChunk ? Mem::K : Mem::Q, r % kChunk, x[n4]);
#pragma unroll
      for (int k = 0; k < kE; ++k) y[n4][k] = 0.f;
    }
    for (int o = 0; o < group; ++o)
#pragma unroll
      for (int n4 = 0; n4 < 4; ++n4) {
        using Vec = std::conditional_t<kE == 4, float4, float2>;
        const Vec z = *reinterpret_cast<const Vec*>(F + (o * own + place[n4]) * Mem::ldF + lane * kE);
        y[n4][0] += z.x;
        y[n4][1] += z.y;
        if constexpr (kE == 4) {
          y[n4][2] += z.z;
          y[n4][3] += z.w;
        }
      }
#pragma unroll
    for (int n4 = 0; n4 < 4; ++n4) {
      dot[n4] = 0.f;
#pragma unroll
      for (int k = 0; k < kE; ++k) dot[n4] = fmaf(x[n4][k], y[n4][k], dot[n4]);
    }
#pragma unroll
    for (int n4 = 0; n4 < 4; ++n4) dot[n4] = lanes_sum(dot[n4]);
#pragma unroll
    for (int n4 = 0; n4 < 4; ++n4) {
      const int r = hg * own + place[n4], i = r % kChunk;
      if (p0 + n4 * kControl >= most || i >= rows || !in) continue;
      const bool of_k = r >= kChunk;
      const float len = of_k ? sh.rk[i] : sh.rq[i] * shorter, by = -len * len * dot[n4];
#pragma unroll
      for (int k = 0; k < kE; ++k) y[n4][k] = fmaf(by, x[n4][k], y[n4][k]);
      I* to = reinterpret_cast<I*>(of_k ? a.dk : a.dq) + (start + i * width);
      if constexpr (kE == 4) *reinterpret_cast<uint2*>(to) = raw_down<I, uint2>(y[n4]);
      else *reinterpret_cast<uint32_t*>(to) = raw_down<I, uint32_t>(y[n4]);
    }
  }
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

template <typename I, int DK, int DV>
void inputs(const DeltaBwd& a, cudaStream_t s) {
  constexpr int bytes = InputsMem<I, DK, DV>::kBytes + (int)sizeof(InputsShared);
  static_assert(bytes <= 227 * 1024, "shared memory");
  cudaFuncSetAttribute(inputs_kernel<I, DK, DV>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.d.B * a.d.H) * a.d.chunks);
  cfg.blockDim = dim3(kWorkers + 32);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = a.d.H / a.d.Hk;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, inputs_kernel<I, DK, DV>, a);
}

template <typename I>
void inputs_of(const DeltaBwd& a, cudaStream_t s) {
  if (a.d.slice == 64) return a.d.dk <= 64 ? inputs<I, 64, 64>(a, s) : inputs<I, 128, 64>(a, s);
  if constexpr (kParts<I> == 1)
    if (a.d.dk > 64) return inputs<I, 128, 128>(a, s);
  inputs<I, 64, 128>(a, s);
}

}  // namespace

void delta_inputs(const DeltaBwd& a, cudaStream_t s) {
  if (a.d.B * a.d.chunks > 0) a.d.type == Elem::kBF16 ? inputs_of<bf16>(a, s) : inputs_of<__half>(a, s);
  gates_kernel<<<a.d.H, 256, 0, s>>>(a);
}

}  // namespace bw
