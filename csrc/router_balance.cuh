// Balance loss of an expert router (router_balance.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "elem.cuh"

namespace bw {

constexpr int kMaxExperts = 1024;

// Router logits (G, N, E), contiguous along E; every group has a loss of its own.
struct BalanceArgs {
  const void* x;
  Elem type;
  long long sg, sn;  // element strides of the group and token axes
  int G, N, E, K;
  const int64_t* ids;   // (G, N, K) chosen experts, or null: the K largest logits, the lowest index where they tie
  const uint8_t* mask;  // (G, N) tokens that count, or null: all
  float z_coef;
  int chunks;           // CTAs of one group
  float* part;          // (G, chunks, E + 1): sums of probabilities, then of squared log-sum-exps
  int* part_count;      // (G, chunks, E + 1): choices, then tokens that count
  float* loss;          // (G)
  int64_t* counts;      // (G, E)
  float* share;         // (G, E + 1): E times the choices of each expert per token, less K; then 1 / tokens
  int* err;
};

struct BalanceGradArgs {
  BalanceArgs f;
  const float* g_loss;  // (G), stride below
  long long g_stride;
  void* out;            // (G, N, E) contiguous
};

// CTAs of one group in the forward.
int balance_chunks(const BalanceArgs& a);
void balance_fwd(const BalanceArgs& a, cudaStream_t s);
void balance_bwd(const BalanceGradArgs& a, cudaStream_t s);

}  // namespace bw
