// Losses over the log-probabilities of chosen tokens, from logits (logit_loss.cu):
// a preference loss over pairs of sequences and a clipped policy loss with a KL term.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "elem.cuh"

namespace bw {

enum class PairLoss : int { kSigmoid = 0, kHinge = 1, kIpo = 2 };
enum class TokenMean : int { kTokens = 0, kSequences = 1, kSum = 2 };

// Logits (B, T, V) with a contiguous last axis and any other strides; labels (B, T) contiguous.
struct LogitRows {
  const void* x;
  long long sb, st;  // element strides of the batch and token axes
  Elem type;
  int B, T, V;
  const int64_t* labels;
  int64_t ignore;
  float inv_temp;
  int* err;  // the device's error word, set where a label is outside [0, V) and not `ignore`
};

// What a row's softmax needs again: exp2((x - m) * c) * inv_s is a probability, c = log2(e) / temperature.
struct RowStat {
  float m, inv_s;
};

struct PreferenceArgs {
  LogitRows rows;
  const float* ref;  // (B): the reference model's log-probability of each sequence
  float* logp_tok;   // (B, T) workspace
  RowStat* stats;    // (B, T)
  float* logps;      // (B)
  float* loss;       // (P) losses of the pairs, or (1)
  float* pair_loss;  // (P) workspace when reduced
  float* dseq;       // (B): d loss / d logps
  float* scale;      // (B): 1, or 1 / tokens when log-probabilities are averaged
  unsigned* ticket;
  PairLoss kind;
  float beta, smoothing, weight;  // weight: 1 / P (mean) or 1
  bool average, reduced;
};

struct PolicyArgs {
  LogitRows rows;
  const float *adv, *old_logps, *ref_logps;  // adv (B, T) or (B); old (B, T) or null; ref (B, T) or null
  bool adv_per_token;
  float clip_lo, clip_hi, kl_coef;
  TokenMean mean;
  float* logps;        // (B, T)
  RowStat* stats;      // (B, T)
  float* dtok;         // (B, T): d loss / d logps
  float4* tok;         // (B, T) workspace: loss, kl, clipped, unused
  double* seq;         // (B, 4) workspace
  int* count;          // (B + 1): tokens of each sequence that count, and of all where there are more than a warp's
  unsigned* ticket;
  float *loss, *kl, *clipped;  // (1) each
  void* grad;          // like the logits, or null: no gradient now
  long long gsb, gst;
};

// d loss / d logits = coef (onehot - softmax) / temperature,
// coef = (g_loss * d + g_logps) * scale with d, g_logps per sequence or per row.
struct LogitGradArgs {
  LogitRows rows;
  const RowStat* stats;
  const float* d;
  const float* g_loss;   // (1), or (P) with g_loss_mod = P; null: no gradient of the loss
  int g_loss_mod;
  const float* g_logps;  // null: none
  const float* scale;    // (B) or null
  bool per_row;
  void* out;
  long long osb, ost;
  // `out` has the gradient for g_loss = 1 already, with zeros in the rows that do not count: g_loss is one number, and
  // there is no g_logps.
  bool unit_grad;
};

void preference_fwd(const PreferenceArgs& a, cudaStream_t s);
// Returns the kernels launched.
int policy_fwd(const PolicyArgs& a, cudaStream_t s);
void logit_grad(const LogitGradArgs& a, cudaStream_t s);

}  // namespace bw
