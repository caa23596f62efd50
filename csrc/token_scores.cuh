// Log-probabilities of chosen tokens, entropies and best alternatives of rows of logits (token_scores.cu).
#pragma once

#include "logit_loss.cuh"

namespace bw {

constexpr int kMostTop = 32;  // alternatives of a row: one for each lane of a warp

// What the backward needs of a row beside its logits: the maximum, log2 of the sum, the entropy.
struct ScoreStat {
  float base, log2_s, entropy;
};

struct ScoreArgs {
  LogitRows rows;
  int top;
  float *logps, *entropy;  // (B, T)
  ScoreStat* stats;        // (B, T), or null without a gradient to come
  float* top_logps;        // (B, T, top)
  int64_t* top_ids;
};

struct ScoreGradArgs {
  LogitRows rows;
  const ScoreStat* stats;
  const float *g_logps, *g_entropy;  // (B, T) or null
  void* out;
  long long osb, ost;
};

void token_scores_fwd(const ScoreArgs& a, cudaStream_t s);
void token_scores_bwd(const ScoreGradArgs& a, cudaStream_t s);

}  // namespace bw
