// What the operators' C++ entry points share: checks of arguments and what their autograd nodes do alike.
#pragma once

#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <memory>
#include <optional>
#include <string>
#include <vector>

#include "logit_loss.cuh"

namespace bw::entry {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients are the kernels' own results: they carry no graph. Under create_graph they come with a node that raises
// when something is differentiated through them.
inline variable_list once(variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads) {
    if (!g.defined()) continue;
    g = g.detach().requires_grad_();
    auto node = std::make_shared<torch::autograd::DelayedError>(
        std::string("the gradient of ") + name + " cannot be differentiated", 1);
    g = (*node)({g})[0];
  }
  return grads;
}

// A gradient that a kernel reads as a dense array, or nothing.
inline OptTensor dense(const Tensor& g) { return g.defined() ? OptTensor(g.contiguous()) : std::nullopt; }

inline bw::Elem elem_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case torch::kBFloat16:
      return bw::Elem::kBF16;
    case torch::kHalf:
      return bw::Elem::kF16;
    case torch::kFloat32:
      return bw::Elem::kF32;
    default:
      TORCH_CHECK_TYPE(false, name, " must be bfloat16, float16 or float32, got ", t.scalar_type());
  }
}

inline void check_like(const Tensor& t, const char* name, torch::ScalarType type, const Tensor& with) {
  TORCH_CHECK(t.is_cuda() && t.device() == with.device(), name, " must be on ", with.device());
  TORCH_CHECK_TYPE(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

inline const float* floats(const OptTensor& t) { return t.has_value() ? t->data_ptr<float>() : nullptr; }

inline bw::LogitRows logit_rows(const Tensor& logits, const Tensor& labels, int64_t ignore, double temperature,
                         const Tensor& err) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 3, "logits must be a (B, T, V) CUDA tensor");
  const int64_t B = logits.size(0), T = logits.size(1), V = logits.size(2);
  TORCH_CHECK(V >= 1 && V < (int64_t(1) << 30), "logits: the vocabulary must have 1 to 2^30 - 1 entries");
  TORCH_CHECK(V == 1 || logits.stride(2) == 1 || logits.numel() == 0, "logits must be contiguous along the vocabulary");
  TORCH_CHECK(B * T < (int64_t(1) << 31), "logits: at most 2^31 - 1 rows");
  check_like(labels, "labels", torch::kInt64, logits);
  TORCH_CHECK(labels.dim() == 2 && labels.size(0) == B && labels.size(1) == T, "labels must be (B, T)");
  check_like(err, "err", torch::kInt32, logits);
  return bw::LogitRows{logits.data_ptr(),          logits.stride(0), logits.stride(1), elem_of(logits, "logits"),
                       (int)B,                     (int)T,           (int)V,           labels.data_ptr<int64_t>(),
                       ignore,                     (float)(1.0 / temperature),         err.data_ptr<int>()};
}

// Memory for the gradient of `logits`. Its rows start at the same offset within 16 bytes as the rows of the logits
// wherever those do not overlap, so that both sides move whole vectors.
inline Tensor grad_like(const Tensor& logits) {
  const int64_t n = 16 / logits.element_size(), V = logits.size(2);
  const auto shift = (int64_t)(reinterpret_cast<uintptr_t>(logits.data_ptr()) % 16) / logits.element_size();
  if (logits.is_contiguous() && shift == 0) return torch::empty(logits.sizes(), logits.options());
  const bool even = V % n == 0;
  if (even && shift == 0 && logits.stride(0) % n == 0 && logits.stride(1) % n == 0)
    return torch::empty(logits.sizes(), logits.options());
  const int64_t B = logits.size(0), T = logits.size(1), sb = logits.stride(0), st = logits.stride(1);
  const bool apart = (T <= 1 || st >= V) && (B <= 1 || sb >= V) &&
                     (T <= 1 || B <= 1 || sb >= (T - 1) * st + V || st >= (B - 1) * sb + V);
  if (!apart || logits.numel() == 0) return torch::empty(logits.sizes(), logits.options());
  const int64_t span = (B - 1) * sb + (T - 1) * st + V + shift;
  if (span > 2 * logits.numel() + n) return torch::empty(logits.sizes(), logits.options());
  return torch::empty({span}, logits.options()).as_strided(logits.sizes(), logits.strides(), shift);
}

// The device's error word is no saved variable of a node: clearing it between a forward and its backward, which is what
// reporting an error does, must not read as a change of the forward's inputs.
inline Tensor error_word(AutogradContext* ctx) { return ctx->saved_data["err"].toTensor(); }

// Without a gradient to come there is no node.
inline bool wants_grad(const Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }

// The kernels read memory and have no forward-mode derivative: a tensor of a functional transform, which has no memory, is
// turned away, and so is one with a tangent, which would be lost without a word.
inline void plain(const Tensor& t, const char* name) {
  TORCH_CHECK_NOT_IMPLEMENTED(t.has_storage(), name, " has no memory of its own (a functional transform, a sparse tensor)");
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode(),
                              "forward-mode derivatives are not implemented on the GPU: ", name, " has a tangent");
}

inline void plain(const OptTensor& t, const char* name) {
  if (t.has_value()) plain(*t, name);
}

inline bool whole_numbers(const Tensor& t) { return at::isIntegralType(t.scalar_type(), false); }

inline void take_logits(Tensor& logits, Tensor& labels) {
  plain(logits, "logits");
  plain(labels, "labels");
  TORCH_CHECK_VALUE(logits.dim() == 3 && at::isFloatingType(logits.scalar_type()), "logits must be floating (B, T, V), got ",
                    logits.scalar_type());
  TORCH_CHECK_VALUE(labels.dim() == 2 && labels.size(0) == logits.size(0) && labels.size(1) == logits.size(1) &&
                        whole_numbers(labels),
                    "labels must be whole numbers (B, T), got ", labels.scalar_type());
  TORCH_CHECK_VALUE(logits.size(2) > 0, "logits need a vocabulary of at least one entry");
  TORCH_CHECK_VALUE(labels.device() == logits.device(), "labels are on ", labels.device(), ", logits on ", logits.device());
  if (logits.stride(2) != 1) logits = logits.contiguous();
  labels = labels.to(torch::kInt64).contiguous();
}

inline Tensor constant(const Tensor& t, const char* name) {
  plain(t, name);
  TORCH_CHECK_VALUE(!t.requires_grad(), name, " is a constant of the loss: detach it");
  return t.to(torch::kFloat32).contiguous();
}

}  // namespace bw::entry
