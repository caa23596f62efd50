// Bindings of the operators of trajectory training: the AdamW step of many tensors and token scores. Arguments are
// checked here and autograd functions are C++ for the reasons that post_training.cpp gives.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include <atomic>
#include <cmath>
#include <unordered_set>

#include "adamw.cuh"
#include "entry.h"
#include "token_scores.cuh"

namespace {

using namespace bw::entry;

std::atomic<int64_t> launches{0};

// ---------------------------------------------------------------- AdamW
bool at_multiple(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

void moment_like(const Tensor& t, const char* name, torch::ScalarType type, const Tensor& p) {
  TORCH_CHECK_VALUE(t.device() == p.device() && t.sizes() == p.sizes() && t.strides() == p.strides(), name,
                    " must have the shape, strides and device of its parameter");
  TORCH_CHECK_TYPE(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
}

void adamw_step(const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const std::vector<Tensor>& exp_avgs,
                const std::vector<Tensor>& exp_avg_sqs, const std::optional<std::vector<Tensor>>& scales, int64_t step,
                double lr, double beta1, double beta2, double eps, double weight_decay, bool maximize) {
  const size_t count = params.size();
  TORCH_CHECK_VALUE(grads.size() == count && exp_avgs.size() == count && exp_avg_sqs.size() == count &&
                        (!scales.has_value() || scales->size() == count),
                    "every parameter needs a gradient and both moments (and scales of both, or of none)");
  if (count == 0) return;
  const bool bits8 = scales.has_value();
  const auto moment = bits8 ? torch::kFloat8_e4m3fn : torch::kFloat32;
  std::unordered_set<const void*> seen;
  seen.reserve(2 * count);
  std::vector<Tensor> held;  // gradients laid out like their parameters
  for (size_t i = 0; i < count; ++i) {
    const Tensor &p = params[i], &g = grads[i];
    for (const auto& [t, name] : {std::pair<const Tensor&, const char*>{p, "a parameter"},
                                  {g, "a gradient"}, {exp_avgs[i], "exp_avg"}, {exp_avg_sqs[i], "exp_avg_sq"}}) {
      TORCH_CHECK_NOT_IMPLEMENTED(t.layout() == torch::kStrided, name, " must be dense, got ", t.layout());
      plain(t, name);
    }
    TORCH_CHECK_VALUE(p.is_cuda() && p.device() == params[0].device(), "parameters must be on one CUDA device");
    elem_of(p, "parameters");
    TORCH_CHECK_VALUE(g.device() == p.device() && g.sizes() == p.sizes(), "a gradient must have its parameter's shape and device");
    TORCH_CHECK_TYPE(g.scalar_type() == p.scalar_type() || g.scalar_type() == torch::kFloat32,
                     "a gradient must be its parameter's type or float32, got ", g.scalar_type());
    TORCH_CHECK_VALUE(p.is_non_overlapping_and_dense(), "parameters must be dense in memory, in any order of their axes");
    moment_like(exp_avgs[i], "exp_avg", moment, p);
    moment_like(exp_avg_sqs[i], "exp_avg_sq", moment, p);
    if (bits8) {
      const Tensor& s = (*scales)[i];
      plain(s, "scales");
      TORCH_CHECK_VALUE(s.device() == p.device() && s.scalar_type() == torch::kFloat32 && s.is_contiguous() && s.dim() == 2 &&
                            s.size(0) == 2 && s.size(1) == (p.numel() + bw::kMomentBlock - 1) / bw::kMomentBlock,
                        "scales must be contiguous float32 (2, blocks of ", std::to_string(bw::kMomentBlock), " elements)");
    }
    if (p.numel() > 0)
      TORCH_CHECK_VALUE(seen.insert(p.data_ptr()).second, "a parameter is given twice");
  }
  bw::AdamwTable table;
  table.beta1 = (float)beta1;
  table.beta2 = (float)beta2;
  table.one_beta1 = (float)(1 - beta1);
  table.one_beta2 = (float)(1 - beta2);
  table.keep = (float)(1 - lr * weight_decay);
  table.size = (float)(lr / (1 - std::pow(beta1, (double)step)));
  table.inv_root2 = (float)(1 / std::sqrt(1 - std::pow(beta2, (double)step)));
  table.eps = (float)eps;
  table.sign = maximize ? -1.f : 1.f;
  const c10::cuda::CUDAGuard guard(params[0].device());
  const auto stream = at::cuda::getCurrentCUDAStream();
  using bw::Elem;
  for (const auto& [pt, gt] : {std::pair<Elem, Elem>{Elem::kBF16, Elem::kBF16}, {Elem::kBF16, Elem::kF32},
                               {Elem::kF16, Elem::kF16}, {Elem::kF16, Elem::kF32}, {Elem::kF32, Elem::kF32}}) {
    table.count = 0;
    table.chunks = 0;
    const auto flush = [&] {
      if (table.count == 0) return;
      bw::adamw_step(table, pt, gt, bits8, stream);
      C10_CUDA_KERNEL_LAUNCH_CHECK();
      ++launches;
      table.count = 0;
      table.chunks = 0;
    };
    for (size_t i = 0; i < count; ++i) {
      const Tensor& p = params[i];
      if (p.numel() == 0 || elem_of(p, "") != pt || elem_of(grads[i], "") != gt) continue;
      Tensor g = grads[i];
      if (g.strides() != p.strides()) {
        g = torch::empty_strided(p.sizes(), p.strides(), g.options());
        g.copy_(grads[i].detach());
        held.push_back(g);
      }
      bw::AdamwTensor& t = table.t[table.count];
      t = bw::AdamwTensor{p.data_ptr(),  g.data_ptr(),
                          exp_avgs[i].data_ptr(), exp_avg_sqs[i].data_ptr(),
                          bits8 ? (*scales)[i].data_ptr<float>() : nullptr, p.numel(), table.chunks, 0u};
      t.aligned = at_multiple(t.p, 16) && at_multiple(t.g, 16) && at_multiple(t.m, bits8 ? 8 : 16) && at_multiple(t.v, bits8 ? 8 : 16);
      const int64_t chunks = (p.numel() + bw::kAdamwChunk - 1) / bw::kAdamwChunk;
      TORCH_CHECK_VALUE(chunks < (int64_t(1) << 30), "a parameter has more than 2^43 elements");
      table.chunks += (unsigned)chunks;
      if (++table.count == bw::kAdamwTensors || table.chunks >= (1u << 30)) flush();
    }
    flush();
  }
  // What autograd saved of these tensors is no longer theirs.
  for (size_t i = 0; i < count; ++i)
    for (const Tensor* t : {&params[i], &exp_avgs[i], &exp_avg_sqs[i]})
      if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  if (bits8)
    for (const Tensor& t : *scales)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// ---------------------------------------------------------------- token scores
// {logps, entropy, top_logps, top_ids, statistics of the rows (with `keep`)}
variable_list scores_fwd(const Tensor& logits, const Tensor& labels, int64_t top, double temperature, int64_t ignore,
                         const Tensor& err, bool keep) {
  const c10::cuda::CUDAGuard guard(logits.device());
  bw::ScoreArgs a;
  a.rows = logit_rows(logits, labels, ignore, temperature, err);
  const int64_t B = a.rows.B, T = a.rows.T;
  const auto f32 = logits.options().dtype(torch::kFloat32);
  auto logps = torch::empty({B, T}, f32), entropy = torch::empty({B, T}, f32), top_logps = torch::empty({B, T, top}, f32);
  auto ids = torch::empty({B, T, top}, logits.options().dtype(torch::kInt64));
  auto stats = torch::empty({keep ? B * T * 3 : 0}, f32);
  a.top = (int)top;
  a.logps = logps.data_ptr<float>();
  a.entropy = entropy.data_ptr<float>();
  a.stats = keep ? reinterpret_cast<bw::ScoreStat*>(stats.data_ptr<float>()) : nullptr;
  a.top_logps = top_logps.data_ptr<float>();
  a.top_ids = ids.data_ptr<int64_t>();
  bw::token_scores_fwd(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  ++launches;
  return {logps, entropy, top_logps, ids, stats};
}

Tensor scores_bwd(const Tensor& logits, const Tensor& labels, const Tensor& stats, const OptTensor& g_logps,
                  const OptTensor& g_entropy, double temperature, int64_t ignore, const Tensor& err) {
  const c10::cuda::CUDAGuard guard(logits.device());
  bw::ScoreGradArgs a;
  a.rows = logit_rows(logits, labels, ignore, temperature, err);
  a.stats = reinterpret_cast<const bw::ScoreStat*>(stats.data_ptr<float>());
  a.g_logps = floats(g_logps);
  a.g_entropy = floats(g_entropy);
  auto out = grad_like(logits);
  a.out = out.data_ptr();
  a.osb = out.stride(0);
  a.ost = out.stride(1);
  bw::token_scores_bwd(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  ++launches;
  return out;
}

struct TokenScores : torch::autograd::Function<TokenScores> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, int64_t top,
                               double temperature, int64_t ignore, const Tensor& err) {
    auto out = scores_fwd(logits, labels, top, temperature, ignore, err, true);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({out[2], out[3]});
    ctx->save_for_backward({logits, labels, out[4]});
    ctx->saved_data["err"] = err;
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore"] = ignore;
    out.pop_back();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(6);
    if (!g[0].defined() && !g[1].defined()) return out;
    const auto s = ctx->get_saved_variables();
    out[0] = scores_bwd(s[0], s[1], s[2], dense(g[0]), dense(g[1]), ctx->saved_data["temperature"].toDouble(),
                        ctx->saved_data["ignore"].toInt(), error_word(ctx));
    return once(std::move(out), "token_scores");
  }
};

variable_list token_scores(Tensor logits, Tensor labels, int64_t top, double temperature, int64_t ignore, Tensor err) {
  take_logits(logits, labels);
  TORCH_CHECK_VALUE(top >= 0 && top <= bw::kMostTop && top <= logits.size(2), "top_k must be between 0 and ", std::to_string(bw::kMostTop),
                    " and no more than the vocabulary");
  TORCH_CHECK_VALUE(temperature > 0 && std::isfinite(temperature), "temperature must be positive");
  if (wants_grad(logits)) return TokenScores::apply(logits, labels, top, temperature, ignore, err);
  auto out = scores_fwd(logits, labels, top, temperature, ignore, err, false);
  out.pop_back();
  return out;
}

}  // namespace

namespace bw {

void register_trajectory(pybind11::module_& m) {
  m.def("adamw_step", &::adamw_step, "AdamW step of many tensors, moments in 32 or 8 bits");
  m.def("token_scores", &::token_scores, "log-probabilities, entropies and best alternatives from logits");
  m.def("trajectory_launches", [] { return launches.load(); }, "kernels that these functions launched");
}

}  // namespace bw
