// Bindings of the post-training operators: preference and policy losses from logits, the
// router's balance loss, and head norms with rotation.
//
// Their autograd functions are C++: a backward node written in Python takes the interpreter
// lock from the engine's thread, which cost more than the kernels of a small call (forward and
// backward of 96 logit rows on one B200: 111 us with Python nodes and checks, 87 us with these nodes, 70 us with the checks
// here too; 45 us of it are the engine's).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <initializer_list>
#include <string>

#include "entry.h"
#include "qk_norm.cuh"
#include "router_balance.cuh"

namespace {

using namespace bw::entry;

std::atomic<int64_t> launches{0};

// The float workspace of a preference loss: [stats 2 R | d (B) | scale (B) | token log-probabilities R | pair losses P | ticket].
variable_list preference_fwd(const Tensor& logits, const Tensor& labels, const Tensor& ref, int64_t kind, double beta,
                             double smoothing, bool average, int64_t reduction, int64_t ignore, const Tensor& err) {
  const c10::cuda::CUDAGuard guard(logits.device());
  bw::PreferenceArgs a;
  a.rows = logit_rows(logits, labels, ignore, 1.0, err);
  const int64_t B = a.rows.B, P = B / 2, R = B * a.rows.T;
  TORCH_CHECK(B >= 2 && B % 2 == 0, "a preference loss needs an even number of sequences: chosen, then rejected");
  check_like(ref, "ref_logps", torch::kFloat32, logits);
  TORCH_CHECK(ref.numel() == B, "ref_logps must be (B)");
  const auto f32 = logits.options().dtype(torch::kFloat32);
  auto ws = torch::empty({2 * R + 2 * B + R + P + 1}, f32);
  auto logps = torch::empty({B}, f32);
  auto loss = reduction == 0 ? torch::empty({P}, f32) : torch::empty({}, f32);
  float* w = ws.data_ptr<float>();
  a.ref = ref.data_ptr<float>();
  a.stats = reinterpret_cast<bw::RowStat*>(w);
  a.dseq = w + 2 * R;
  a.scale = a.dseq + B;
  a.logp_tok = a.scale + B;
  a.pair_loss = a.logp_tok + R;
  a.ticket = reinterpret_cast<unsigned*>(a.pair_loss + P);
  a.logps = logps.data_ptr<float>();
  a.loss = loss.data_ptr<float>();
  a.kind = (bw::PairLoss)kind;
  a.beta = (float)beta;
  a.smoothing = (float)smoothing;
  a.weight = reduction == 1 ? 1.f / (float)P : 1.f;
  a.average = average;
  a.reduced = reduction != 0;
  bw::preference_fwd(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {loss, logps, ws};
}

Tensor preference_bwd(const Tensor& logits, const Tensor& labels, const Tensor& ws, const OptTensor& g_loss,
                      const OptTensor& g_logps, int64_t ignore, const Tensor& err) {
  const c10::cuda::CUDAGuard guard(logits.device());
  bw::LogitGradArgs a;
  a.rows = logit_rows(logits, labels, ignore, 1.0, err);
  const int64_t B = a.rows.B, R = B * a.rows.T;
  check_like(ws, "workspace", torch::kFloat32, logits);
  TORCH_CHECK(ws.numel() >= 3 * R + 2 * B, "workspace is too small");
  if (g_loss.has_value()) {
    check_like(*g_loss, "loss gradient", torch::kFloat32, logits);
    TORCH_CHECK(g_loss->dim() == 0 || g_loss->numel() == B / 2, "loss gradient must be a scalar or (P)");
  }
  if (g_logps.has_value()) {
    check_like(*g_logps, "logps gradient", torch::kFloat32, logits);
    TORCH_CHECK(g_logps->numel() == B, "logps gradient must be (B)");
  }
  auto out = grad_like(logits);
  const float* w = ws.data_ptr<float>();
  a.stats = reinterpret_cast<const bw::RowStat*>(w);
  a.d = w + 2 * R;
  a.scale = a.d + B;
  a.g_loss = floats(g_loss);
  a.g_loss_mod = g_loss.has_value() && g_loss->dim() > 0 ? (int)(B / 2) : 0;
  a.g_logps = floats(g_logps);
  a.per_row = false;
  a.unit_grad = false;
  a.out = out.data_ptr();
  a.osb = out.stride(0);
  a.ost = out.stride(1);
  bw::logit_grad(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

// The float workspace of a policy loss: [stats 2 R | d R | (4 R of tokens) | sums of sequences 8 B | token counts B, all | ticket].
// With want_grad the result's last tensor is the gradient for a loss gradient of 1.
variable_list policy_fwd(const Tensor& logits, const Tensor& labels, const Tensor& adv, const OptTensor& old_logps,
                         const OptTensor& ref_logps, double clip_lo, double clip_hi, double kl_coef, double temperature,
                         int64_t mean, int64_t ignore, const Tensor& err, bool want_grad) {
  const c10::cuda::CUDAGuard guard(logits.device());
  bw::PolicyArgs a;
  a.rows = logit_rows(logits, labels, ignore, temperature, err);
  const int64_t B = a.rows.B, T = a.rows.T, R = B * T;
  TORCH_CHECK(B >= 1, "a policy loss needs at least one sequence");
  check_like(adv, "advantages", torch::kFloat32, logits);
  TORCH_CHECK((adv.dim() == 1 && adv.size(0) == B) || (adv.dim() == 2 && adv.size(0) == B && adv.size(1) == T),
              "advantages must be (B) or (B, T)");
  for (const auto& [t, name] : {std::pair<const OptTensor&, const char*>{old_logps, "old_logps"}, {ref_logps, "ref_logps"}}) {
    if (!t.has_value()) continue;
    check_like(*t, name, torch::kFloat32, logits);
    TORCH_CHECK(t->dim() == 2 && t->size(0) == B && t->size(1) == T, name, " must be (B, T)");
  }
  const auto f32 = logits.options().dtype(torch::kFloat32);
  const int64_t even = (2 * R + R + 3) / 4 * 4;  // the tokens' float4 start on their boundary
  auto ws = torch::empty({even + 4 * R + 8 * B + B + 2}, f32);
  auto logps = torch::empty({B, T}, f32);
  auto loss = torch::empty({}, f32), kl = torch::empty({}, f32), clipped = torch::empty({}, f32);
  float* w = ws.data_ptr<float>();
  a.adv = adv.data_ptr<float>();
  a.old_logps = floats(old_logps);
  a.ref_logps = floats(ref_logps);
  a.adv_per_token = adv.dim() == 2;
  a.clip_lo = (float)clip_lo;
  a.clip_hi = (float)clip_hi;
  a.kl_coef = (float)kl_coef;
  a.mean = (bw::TokenMean)mean;
  a.logps = logps.data_ptr<float>();
  a.stats = reinterpret_cast<bw::RowStat*>(w);
  a.dtok = w + 2 * R;
  a.tok = reinterpret_cast<float4*>(w + even);
  a.seq = reinterpret_cast<double*>(a.tok + R);
  a.count = reinterpret_cast<int*>(a.seq + 4 * B);
  a.ticket = reinterpret_cast<unsigned*>(a.count + B + 1);
  a.loss = loss.data_ptr<float>();
  a.kl = kl.data_ptr<float>();
  a.clipped = clipped.data_ptr<float>();
  Tensor grad;
  a.grad = nullptr;
  if (want_grad) {
    grad = grad_like(logits);
    a.grad = grad.data_ptr();
    a.gsb = grad.stride(0);
    a.gst = grad.stride(1);
  }
  launches += bw::policy_fwd(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {loss, logps, kl, clipped, ws, grad};
}

// unit_grad: the gradient for a loss gradient of 1, which is given out where that is what the loss has; undefined: none.
Tensor policy_bwd(const Tensor& logits, const Tensor& labels, const Tensor& ws, const OptTensor& g_loss,
                  const OptTensor& g_logps, double temperature, int64_t ignore, const Tensor& err, Tensor unit_grad) {
  const c10::cuda::CUDAGuard guard(logits.device());
  bw::LogitGradArgs a;
  a.rows = logit_rows(logits, labels, ignore, temperature, err);
  const int64_t R = (int64_t)a.rows.B * a.rows.T;
  check_like(ws, "workspace", torch::kFloat32, logits);
  TORCH_CHECK(ws.numel() >= 3 * R, "workspace is too small");
  if (g_loss.has_value()) {
    check_like(*g_loss, "loss gradient", torch::kFloat32, logits);
    TORCH_CHECK(g_loss->numel() == 1, "loss gradient must be a scalar");
  }
  if (g_logps.has_value()) {
    check_like(*g_logps, "logps gradient", torch::kFloat32, logits);
    TORCH_CHECK(g_logps->numel() == R, "logps gradient must be (B, T)");
  }
  a.unit_grad = unit_grad.defined() && g_loss.has_value() && !g_logps.has_value();
  auto out = a.unit_grad ? std::move(unit_grad) : grad_like(logits);
  const float* w = ws.data_ptr<float>();
  a.stats = reinterpret_cast<const bw::RowStat*>(w);
  a.d = w + 2 * R;
  a.scale = nullptr;
  a.g_loss = floats(g_loss);
  a.g_loss_mod = 0;
  a.g_logps = floats(g_logps);
  a.per_row = true;
  a.out = out.data_ptr();
  a.osb = out.stride(0);
  a.ost = out.stride(1);
  bw::logit_grad(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

bw::BalanceArgs balance_args(const Tensor& logits, const OptTensor& ids, const OptTensor& mask, int64_t top_k,
                             double z_coef, const Tensor& err) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 3, "router logits must be a (G, N, E) CUDA tensor");
  bw::BalanceArgs a{};
  const int64_t G = logits.size(0), N = logits.size(1), E = logits.size(2);
  TORCH_CHECK(E >= 1 && E <= bw::kMaxExperts, "router logits: 1 to ", std::to_string(bw::kMaxExperts), " experts");
  TORCH_CHECK(E == 1 || logits.stride(2) == 1 || logits.numel() == 0, "router logits must be contiguous along the experts");
  TORCH_CHECK(top_k >= 1 && top_k <= E, "top_k must be between 1 and the number of experts");
  TORCH_CHECK(G <= 65535, "router logits: at most 65535 groups");
  TORCH_CHECK(N < (int64_t(1) << 31) / (top_k > 8 ? top_k : 8), "router logits: too many tokens in a group");
  a.x = logits.data_ptr();
  a.type = elem_of(logits, "router logits");
  a.sg = logits.stride(0);
  a.sn = logits.stride(1);
  a.G = (int)G;
  a.N = (int)N;
  a.E = (int)E;
  a.K = (int)top_k;
  if (ids.has_value()) {
    check_like(*ids, "expert_ids", torch::kInt64, logits);
    TORCH_CHECK(ids->numel() == G * N * top_k, "expert_ids must be (..., N, top_k)");
    a.ids = ids->data_ptr<int64_t>();
  }
  if (mask.has_value()) {
    check_like(*mask, "mask", torch::kBool, logits);
    TORCH_CHECK(mask->numel() == G * N, "mask must be (..., N)");
    a.mask = reinterpret_cast<const uint8_t*>(mask->data_ptr<bool>());
  }
  a.z_coef = (float)z_coef;
  a.chunks = bw::balance_chunks(a);
  check_like(err, "err", torch::kInt32, logits);
  a.err = err.data_ptr<int>();
  return a;
}

variable_list balance_fwd(const Tensor& logits, const OptTensor& ids, const OptTensor& mask, int64_t top_k, double z_coef,
                          const Tensor& err) {
  const c10::cuda::CUDAGuard guard(logits.device());
  bw::BalanceArgs a = balance_args(logits, ids, mask, top_k, z_coef, err);
  const auto f32 = logits.options().dtype(torch::kFloat32);
  const int64_t cells = (int64_t)a.G * a.chunks * (a.E + 1);
  auto part = torch::empty({2 * cells}, f32);
  auto loss = torch::empty({a.G}, f32), share = torch::empty({a.G, a.E + 1}, f32);
  auto counts = torch::empty({a.G, a.E}, logits.options().dtype(torch::kInt64));
  a.part = part.data_ptr<float>();
  a.part_count = reinterpret_cast<int*>(a.part + cells);
  a.loss = loss.data_ptr<float>();
  a.counts = counts.data_ptr<int64_t>();
  a.share = share.data_ptr<float>();
  if (a.G > 0) bw::balance_fwd(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {loss, counts, share};
}

Tensor balance_bwd(const Tensor& logits, const OptTensor& mask, const Tensor& share, const Tensor& g_loss, int64_t top_k,
                   double z_coef, const Tensor& err) {
  const c10::cuda::CUDAGuard guard(logits.device());
  bw::BalanceGradArgs b;
  b.f = balance_args(logits, std::nullopt, mask, top_k, z_coef, err);
  check_like(share, "share", torch::kFloat32, logits);
  TORCH_CHECK(share.numel() == (int64_t)b.f.G * (b.f.E + 1), "share must be (G, E + 1)");
  TORCH_CHECK(g_loss.is_cuda() && g_loss.scalar_type() == torch::kFloat32 && g_loss.dim() == 1 && g_loss.size(0) == b.f.G,
              "loss gradient must be (G) float32");
  b.f.share = share.data_ptr<float>();
  b.g_loss = g_loss.data_ptr<float>();
  b.g_stride = g_loss.stride(0);
  auto out = torch::empty(logits.sizes(), logits.options());
  b.out = out.data_ptr();
  if (out.numel() > 0) bw::balance_bwd(b, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

bw::HeadTensor head_tensor(const Tensor& x, const Tensor& w, const char* name) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 4, name, " must be a (B, T, H, D) CUDA tensor");
  TORCH_CHECK(x.size(3) == 1 || x.stride(3) == 1 || x.numel() == 0, name, " must be contiguous along the head's elements");
  TORCH_CHECK(w.is_cuda() && w.device() == x.device() && w.dim() == 1 && w.size(0) == x.size(3) && w.is_contiguous(),
              name, " weight must be a contiguous (D) tensor on the same device");
  return bw::HeadTensor{x.data_ptr(), x.stride(0), x.stride(1), x.stride(2), nullptr, w.data_ptr(), (int)x.size(2)};
}

bw::QkNormArgs qk_args(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw, const Tensor& cos,
                       const Tensor& sin, const OptTensor& positions, double eps, const Tensor& err) {
  bw::QkNormArgs a{};
  a.q = head_tensor(q, qw, "q");
  a.k = head_tensor(k, kw, "k");
  TORCH_CHECK(q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3) && q.device() == k.device(),
              "q and k must be (B, T, H, D) with the same B, T and D");
  a.type = elem_of(q, "q");
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type(), "q and k must have one type");
  a.wtype = elem_of(qw, "weights");
  TORCH_CHECK_TYPE(kw.scalar_type() == qw.scalar_type(), "both weights must have one type");
  a.B = (int)q.size(0);
  a.T = (int)q.size(1);
  a.D = (int)q.size(3);
  TORCH_CHECK(a.D >= 2 && a.D % 2 == 0 && a.D <= bw::kMaxHeadDim, "the head dim must be even and at most ",
              std::to_string(bw::kMaxHeadDim));
  check_like(cos, "cos", torch::kFloat32, q);
  check_like(sin, "sin", torch::kFloat32, q);
  TORCH_CHECK(cos.dim() == 2 && sin.sizes() == cos.sizes() && 2 * cos.size(1) <= a.D,
              "cos and sin must be (positions, R / 2) with R at most the head dim");
  a.cos = cos.data_ptr<float>();
  a.sin = sin.data_ptr<float>();
  a.R = (int)(2 * cos.size(1));
  TORCH_CHECK(cos.size(0) < (int64_t(1) << 31), "cos and sin: at most 2^31 - 1 positions");
  a.table = (int)cos.size(0);
  if (positions.has_value()) {
    TORCH_CHECK(positions->is_cuda() && positions->device() == q.device() && positions->scalar_type() == torch::kInt64 &&
                    positions->dim() == 2 && positions->size(0) == a.B && positions->size(1) == a.T,
                "positions must be (B, T) int64 on the same device");
    TORCH_CHECK(a.table > 0 || q.size(0) * q.size(1) == 0, "the tables of angles are empty");
    a.positions = positions->data_ptr<int64_t>();
    a.pb = positions->stride(0);
    a.pt = positions->stride(1);
  } else {
    TORCH_CHECK(a.table >= a.T, "the tables of angles are shorter than the sequence");
  }
  a.eps = (float)eps;
  TORCH_CHECK(q.size(0) * q.size(1) < (int64_t(1) << 31) && q.size(0) * q.size(1) * (q.size(2) + k.size(2)) < (int64_t(1) << 33),
              "q and k: too many heads");
  check_like(err, "err", torch::kInt32, q);
  a.err = err.data_ptr<int>();
  return a;
}

variable_list qk_norm_fwd(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw, const Tensor& cos,
                          const Tensor& sin, const OptTensor& positions, double eps, const Tensor& err) {
  const c10::cuda::CUDAGuard guard(q.device());
  bw::QkNormArgs a = qk_args(q, k, qw, kw, cos, sin, positions, eps, err);
  auto qo = torch::empty(q.sizes(), q.options()), ko = torch::empty(k.sizes(), k.options());
  a.q.out = qo.data_ptr();
  a.k.out = ko.data_ptr();
  bw::qk_norm_fwd(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {qo, ko};
}

void head_grad(const OptTensor& g, const Tensor& x, const char* name, const void*& p, long long& sb, long long& st,
               long long& sh) {
  p = nullptr;
  sb = st = sh = 0;
  if (!g.has_value()) return;
  TORCH_CHECK(g->is_cuda() && g->device() == x.device() && g->sizes() == x.sizes() &&
                  g->scalar_type() == x.scalar_type() && (x.size(3) == 1 || g->stride(3) == 1 || g->numel() == 0),
              "the gradient of ", name, " must be like it, contiguous along the head's elements");
  p = g->data_ptr();
  sb = g->stride(0);
  st = g->stride(1);
  sh = g->stride(2);
}

variable_list qk_norm_bwd(const OptTensor& gq, const OptTensor& gk, const Tensor& q, const Tensor& k, const Tensor& qw,
                          const Tensor& kw, const Tensor& cos, const Tensor& sin, const OptTensor& positions, double eps,
                          const Tensor& err) {
  const c10::cuda::CUDAGuard guard(q.device());
  bw::QkNormGradArgs b{};
  b.f = qk_args(q, k, qw, kw, cos, sin, positions, eps, err);
  head_grad(gq, q, "q", b.gq, b.gqb, b.gqt, b.gqh);
  head_grad(gk, k, "k", b.gk, b.gkb, b.gkt, b.gkh);
  auto dq = torch::empty(q.sizes(), q.options()), dk = torch::empty(k.sizes(), k.options());
  auto dqw = torch::empty(qw.sizes(), qw.options()), dkw = torch::empty(kw.sizes(), kw.options());
  b.f.q.out = dq.data_ptr();
  b.f.k.out = dk.data_ptr();
  b.dqw = dqw.data_ptr();
  b.dkw = dkw.data_ptr();
  bw::qk_norm_blocks(b, &b.q_blocks, &b.k_blocks);
  auto part = torch::empty({(int64_t)(b.q_blocks + b.k_blocks) * b.f.D}, q.options().dtype(torch::kFloat32));
  b.part = part.data_ptr<float>();
  bw::qk_norm_bwd(b, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {dq, dk, dqw, dkw};
}

// ---------------------------------------------------------------- autograd
struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, const Tensor& ref,
                               int64_t kind, double beta, double smoothing, bool average, int64_t reduction,
                               int64_t ignore, const Tensor& err) {
    auto out = preference_fwd(logits, labels, ref, kind, beta, smoothing, average, reduction, ignore, err);
    launches += 2;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, labels, out[2]});
    ctx->saved_data["err"] = err;
    ctx->saved_data["ignore"] = ignore;
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(10);
    if (!g[0].defined() && !g[1].defined()) return out;
    const auto s = ctx->get_saved_variables();
    out[0] = preference_bwd(s[0], s[1], s[2], dense(g[0]), dense(g[1]), ctx->saved_data["ignore"].toInt(), error_word(ctx));
    ++launches;
    return once(std::move(out), "preference_loss");
  }
};

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, const Tensor& adv,
                               const OptTensor& old_logps, const OptTensor& ref_logps, double clip_lo, double clip_hi,
                               double kl_coef, double temperature, int64_t mean, int64_t ignore, const Tensor& err) {
    auto out = policy_fwd(logits, labels, adv, old_logps, ref_logps, clip_lo, clip_hi, kl_coef, temperature, mean,
                          ignore, err, true);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({out[2], out[3]});
    ctx->save_for_backward({logits, labels, out[4]});
    ctx->saved_data["err"] = err;
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["grad"] = out[5];
    return {out[0], out[1], out[2], out[3]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(12);
    if (!g[0].defined() && !g[1].defined()) return out;
    const auto s = ctx->get_saved_variables();
    // The gradient written by the forward is given away once; another backward through the graph computes it again.
    Tensor unit_grad;
    const auto kept = ctx->saved_data.find("grad");
    if (kept != ctx->saved_data.end()) {
      unit_grad = kept->second.toTensor();
      ctx->saved_data.erase(kept);
    }
    out[0] = policy_bwd(s[0], s[1], s[2], dense(g[0]), dense(g[1]), ctx->saved_data["temperature"].toDouble(),
                        ctx->saved_data["ignore"].toInt(), error_word(ctx), std::move(unit_grad));
    ++launches;
    return once(std::move(out), "policy_loss");
  }
};

struct BalanceLoss : torch::autograd::Function<BalanceLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const OptTensor& ids, const OptTensor& mask,
                               int64_t top_k, double z_coef, const Tensor& err) {
    auto out = balance_fwd(logits, ids, mask, top_k, z_coef, err);
    launches += 2;
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({out[1]});
    ctx->save_for_backward({logits, mask.value_or(Tensor()), out[2]});
    ctx->saved_data["err"] = err;
    ctx->saved_data["top_k"] = top_k;
    ctx->saved_data["z"] = z_coef;
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(6);
    if (!g[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    out[0] = balance_bwd(s[0], s[1].defined() ? OptTensor(s[1]) : std::nullopt, s[2], g[0],
                         ctx->saved_data["top_k"].toInt(), ctx->saved_data["z"].toDouble(), error_word(ctx));
    ++launches;
    return once(std::move(out), "router_balance_loss");
  }
};

struct QkNormRope : torch::autograd::Function<QkNormRope> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& qw,
                               const Tensor& kw, const Tensor& cos, const Tensor& sin, const OptTensor& positions,
                               double eps, const Tensor& err) {
    auto out = qk_norm_fwd(q, k, qw, kw, cos, sin, positions, eps, err);
    ++launches;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, qw, kw, cos, sin, positions.value_or(Tensor())});
    ctx->saved_data["err"] = err;
    ctx->saved_data["eps"] = eps;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(9);
    if (!g[0].defined() && !g[1].defined()) return out;
    const auto s = ctx->get_saved_variables();
    const auto row = [](const Tensor& t) {
      return !t.defined() ? OptTensor() : OptTensor(t.stride(-1) == 1 ? t : t.contiguous());
    };
    auto d = qk_norm_bwd(row(g[0]), row(g[1]), s[0], s[1], s[2], s[3], s[4], s[5],
                         s[6].defined() ? OptTensor(s[6]) : std::nullopt, ctx->saved_data["eps"].toDouble(), error_word(ctx));
    launches += 2;
    std::copy(d.begin(), d.end(), out.begin());
    return once(std::move(out), "qk_norm_rope");
  }
};

// ---------------------------------------------------------------- entry points
// The arguments are checked here and not in Python, where the checks took as long as the rest of a small call.

// The place of `name` among the choices.
int64_t choice(const std::string& name, const char* what, std::initializer_list<const char*> of) {
  int64_t k = 0;
  std::string all;
  for (const char* o : of) {
    if (name == o) return k;
    all += (k++ ? ", '" : "'") + std::string(o) + "'";
  }
  TORCH_CHECK_VALUE(false, what, " must be one of ", all, ", got '", name, "'");
}

variable_list preference_loss(Tensor logits, Tensor labels, Tensor ref, const std::string& kind, double beta,
                              double smoothing, bool average, const std::string& reduction, int64_t ignore, Tensor err) {
  take_logits(logits, labels);
  const int64_t B = logits.size(0);
  TORCH_CHECK_VALUE(B >= 2 && B % 2 == 0, "a preference loss needs an even number of sequences (chosen, then rejected)");
  const int64_t kind_at = choice(kind, "kind", {"sigmoid", "hinge", "ipo"});
  const int64_t reduction_at = choice(reduction, "reduction", {"none", "mean", "sum"});
  TORCH_CHECK_VALUE(beta > 0 && std::isfinite(beta), "beta must be positive");
  TORCH_CHECK_VALUE(smoothing >= 0 && smoothing < 0.5 && (smoothing == 0 || kind_at == 0),
                    "label_smoothing must be in [0, 0.5), and 0 unless kind is 'sigmoid'");
  TORCH_CHECK_VALUE(ref.dim() == 1 && ref.size(0) == B, "ref_logps must have one entry for each sequence");
  ref = constant(ref, "ref_logps");
  if (!wants_grad(logits)) {
    auto out = preference_fwd(logits, labels, ref, kind_at, beta, smoothing, average, reduction_at, ignore, err);
    launches += 2;
    return {out[0], out[1]};
  }
  return PreferenceLoss::apply(logits, labels, ref, kind_at, beta, smoothing, average, reduction_at, ignore, err);
}

variable_list policy_loss(Tensor logits, Tensor labels, Tensor adv, OptTensor old_logps, OptTensor ref_logps, double low,
                          double high, double kl_coef, double temperature, const std::string& reduction, int64_t ignore,
                          Tensor err) {
  take_logits(logits, labels);
  const int64_t B = logits.size(0), T = logits.size(1);
  TORCH_CHECK_VALUE(B > 0, "a policy loss needs at least one sequence");
  const auto per_token = [&](const Tensor& t) { return t.dim() == 2 && t.size(0) == B && t.size(1) == T; };
  TORCH_CHECK_VALUE((adv.dim() == 1 && adv.size(0) == B) || per_token(adv), "advantages must be (B,) or (B, T)");
  TORCH_CHECK_VALUE(!old_logps.has_value() || per_token(*old_logps), "old_logps must be (B, T)");
  TORCH_CHECK_VALUE(!ref_logps.has_value() || per_token(*ref_logps), "ref_logps must be (B, T)");
  const int64_t mean = choice(reduction, "reduction", {"token_mean", "sequence_mean", "sum"});
  TORCH_CHECK_VALUE(temperature > 0 && std::isfinite(temperature), "temperature must be positive");
  TORCH_CHECK_VALUE(low >= 0 && low <= 1 && high >= 0, "clip must be (low in [0, 1], high >= 0)");
  TORCH_CHECK_VALUE(kl_coef == 0 || ref_logps.has_value(), "a KL term needs ref_logps");
  adv = constant(adv, "advantages");
  if (old_logps.has_value()) old_logps = constant(*old_logps, "old_logps");
  if (ref_logps.has_value()) ref_logps = constant(*ref_logps, "ref_logps");
  if (!wants_grad(logits)) {
    auto out = policy_fwd(logits, labels, adv, old_logps, ref_logps, 1 - low, 1 + high, kl_coef, temperature, mean, ignore,
                          err, false);
    return {out[0], out[1], out[2], out[3]};
  }
  return PolicyLoss::apply(logits, labels, adv, old_logps, ref_logps, 1 - low, 1 + high, kl_coef, temperature, mean,
                           ignore, err);
}

variable_list balance_loss(Tensor logits, OptTensor ids, OptTensor mask, int64_t top_k, double z_coef, Tensor err) {
  plain(logits, "router logits");
  plain(ids, "expert_ids");
  plain(mask, "mask");
  TORCH_CHECK_VALUE(logits.dim() >= 2 && at::isFloatingType(logits.scalar_type()),
                    "router logits must be floating (..., N, E), got ", logits.scalar_type());
  const auto lead = logits.sizes().slice(0, logits.dim() - 2).vec();
  const int64_t N = logits.size(-2), E = logits.size(-1), G = c10::multiply_integers(lead);
  TORCH_CHECK_VALUE(top_k >= 1 && top_k <= E, "top_k must be between 1 and the number of experts");
  if (ids.has_value()) {
    auto want = logits.sizes().vec();
    want.back() = top_k;
    TORCH_CHECK_VALUE(ids->sizes() == at::IntArrayRef(want) && whole_numbers(*ids),
                      "expert_ids must be whole numbers (..., N, top_k), got ", ids->scalar_type());
    ids = ids->to(torch::kInt64).contiguous();
  }
  if (mask.has_value()) {
    TORCH_CHECK_VALUE(mask->sizes() == logits.sizes().slice(0, logits.dim() - 1), "mask must be (..., N)");
    mask = (mask->scalar_type() == torch::kBool ? *mask : mask->ne(0)).contiguous();
  }
  if (lead.size() != 1) logits = logits.reshape({G, N, E});
  if (logits.stride(2) != 1) logits = logits.contiguous();
  variable_list out;
  if (!wants_grad(logits)) {
    out = balance_fwd(logits, ids, mask, top_k, z_coef, err);
    launches += 2;
    out.pop_back();
  } else {
    out = BalanceLoss::apply(logits, ids, mask, top_k, z_coef, err);
  }
  if (lead.size() != 1) {
    auto cells = lead;
    cells.push_back(E);
    out = {out[0].reshape(lead), out[1].reshape(cells)};
  }
  return out;
}

// A call by a decoder's every layer and token: its arguments are checked here, not in Python.
variable_list qk_norm_rope(Tensor q, Tensor k, Tensor qw, Tensor kw, Tensor cos, Tensor sin, OptTensor positions,
                           double eps, Tensor err) {
  plain(q, "q");
  plain(k, "k");
  plain(qw, "q_weight");
  plain(kw, "k_weight");
  plain(cos, "cos");
  plain(sin, "sin");
  plain(positions, "positions");
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && q.size(0) == k.size(0) && q.size(1) == k.size(1) &&
                        q.size(3) == k.size(3) && q.scalar_type() == k.scalar_type(),
                    "q and k must be (B, T, H, D) of one type with the same B, T and D");
  const int64_t B = q.size(0), T = q.size(1), D = q.size(3);
  TORCH_CHECK_VALUE(qw.dim() == 1 && kw.dim() == 1 && qw.size(0) == D && kw.size(0) == D && qw.scalar_type() == kw.scalar_type(),
                    "both weights must be (D,) of one type");
  TORCH_CHECK_VALUE(cos.dim() == 2 && cos.sizes() == sin.sizes() && 2 * cos.size(1) <= D && D % 2 == 0,
                    "cos and sin must be (positions, R / 2) with R at most D, and D even");
  TORCH_CHECK_VALUE(!cos.requires_grad() && !sin.requires_grad(), "the tables of angles are constants: detach them");
  if (positions.has_value()) {
    const Tensor& p = *positions;
    TORCH_CHECK_VALUE(((p.dim() == 1 && p.size(0) == T) || (p.dim() == 2 && p.size(0) == B && p.size(1) == T)) &&
                          whole_numbers(p),
                      "positions must be whole numbers (T,) or (B, T)");
    positions = p.to(torch::kInt64);
    if (positions->dim() == 1) positions = positions->expand({B, T});
  } else {
    TORCH_CHECK_VALUE(cos.size(0) >= T, "the tables of angles are shorter than the sequence");
  }
  if (q.stride(3) != 1) q = q.contiguous();
  if (k.stride(3) != 1) k = k.contiguous();
  qw = qw.contiguous();
  kw = kw.contiguous();
  cos = cos.to(torch::kFloat32).contiguous();
  sin = sin.to(torch::kFloat32).contiguous();
  if (!wants_grad(q) && !wants_grad(k) && !wants_grad(qw) && !wants_grad(kw)) {
    ++launches;
    return qk_norm_fwd(q, k, qw, kw, cos, sin, positions, eps, err);
  }
  return QkNormRope::apply(q, k, qw, kw, cos, sin, positions, eps, err);
}

}  // namespace

namespace bw {

void register_post_training(pybind11::module_& m) {
  m.def("preference_loss", &::preference_loss, "preference loss of pairs of sequences from logits");
  m.def("policy_loss", &::policy_loss, "clipped policy loss with a KL term from logits");
  m.def("balance_loss", &::balance_loss, "router balance loss and per-expert counts");
  m.def("qk_norm_rope", &::qk_norm_rope, "RMS norm of q and k heads with rotation by position");
  m.def("post_training_launches", [] { return launches.load(); }, "kernels that these functions launched");
}

}  // namespace bw
