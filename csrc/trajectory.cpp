// Bindings of the operators of trajectory training: the AdamW step of many tensors, token scores and the gated delta rule. Arguments are
// checked here and autograd functions are C++ for the reasons that post_training.cpp gives.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include <atomic>
#include <cmath>
#include <unordered_set>

#include "adamw.cuh"
#include "delta_rule.cuh"
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
  seen.reserve(4 * count);
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
    if (p.numel() > 0) {
      for (const Tensor* t : {&p, &exp_avgs[i], &exp_avg_sqs[i]})
        TORCH_CHECK_VALUE(seen.insert(t->data_ptr()).second, "a parameter or a moment is given twice");
      TORCH_CHECK_VALUE(!bits8 || seen.insert((*scales)[i].data_ptr()).second, "scales are given twice");
    }
  }
  bw::AdamwTable<bw::kAdamwMany> table;
  table.s.beta1 = (float)beta1;
  table.s.beta2 = (float)beta2;
  table.s.one_beta1 = (float)(maximize ? beta1 - 1 : 1 - beta1);
  table.s.one_beta2 = (float)(1 - beta2);
  table.s.keep = (float)(1 - lr * weight_decay);
  table.s.size = (float)(lr / (1 - std::pow(beta1, (double)step)));
  table.s.inv_root2 = (float)(1 / std::sqrt(1 - std::pow(beta2, (double)step)));
  table.s.eps = (float)eps;
  const c10::cuda::CUDAGuard guard(params[0].device());
  const auto stream = at::cuda::getCurrentCUDAStream();
  using bw::Elem;
  for (const auto& [pt, gt] : {std::pair<Elem, Elem>{Elem::kBF16, Elem::kBF16}, {Elem::kBF16, Elem::kF32},
                               {Elem::kF16, Elem::kF16}, {Elem::kF16, Elem::kF32}, {Elem::kF32, Elem::kF32}}) {
    int64_t total = 0;
    for (size_t i = 0; i < count; ++i)
      if (elem_of(params[i], "") == pt && elem_of(grads[i], "") == gt) total += params[i].numel();
    table.s.chunk = bw::adamw_chunk(total, bits8);
    table.s.count = 0;
    table.s.chunks = 0;
    const auto flush = [&] {
      if (table.s.count == 0) return;
      bw::adamw_step(table, pt, gt, bits8, stream);
      C10_CUDA_KERNEL_LAUNCH_CHECK();
      ++launches;
      table.s.count = 0;
      table.s.chunks = 0;
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
      bw::AdamwTensor& t = table.t[table.s.count];
      t = bw::AdamwTensor{p.data_ptr(), g.data_ptr(), exp_avgs[i].data_ptr(), exp_avg_sqs[i].data_ptr(),
                          bits8 ? (*scales)[i].data_ptr<float>() : nullptr, p.numel()};
      const size_t of_moments = bits8 ? 8 : 16;
      if (!at_multiple(t.p, 16) || !at_multiple(t.g, 16) || !at_multiple(t.m, of_moments) || !at_multiple(t.v, of_moments)) t.n = -t.n;
      table.first[table.s.count] = table.s.chunks;
      const int64_t chunks = (p.numel() + table.s.chunk - 1) / table.s.chunk;
      TORCH_CHECK_VALUE(chunks < (int64_t(1) << 30), "a parameter has 2^41 elements or more");
      table.s.chunks += (unsigned)chunks;
      if (++table.s.count == bw::kAdamwMany || table.s.chunks >= (1u << 30)) flush();
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

// ---------------------------------------------------------------- gated delta rule
struct DeltaIn {
  Tensor q, k, v, a, b, a_log, dt_bias;
};

bw::HeadRows head_rows(const Tensor& t) {
  return bw::HeadRows{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

// Rows on 16-byte boundaries.
bool rows_aligned(const Tensor& t) {
  const int64_t n = 16 / t.element_size();
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1 && t.stride(i) % n != 0) return false;
  return at_multiple(t.data_ptr(), 16);
}

bw::DeltaDims delta_dims(const DeltaIn& x, double scale) {
  bw::DeltaDims d;
  d.B = (int)x.q.size(0);
  d.T = (int)x.q.size(1);
  d.Hk = (int)x.q.size(2);
  d.dk = (int)x.q.size(3);
  d.H = (int)x.v.size(2);
  d.dv = (int)x.v.size(3);
  d.chunks = (d.T + bw::kChunk - 1) / bw::kChunk;
  d.type = elem_of(x.q, "q");
  d.scale = (float)scale;
  d.wide = rows_aligned(x.q) && rows_aligned(x.k);
  d.slice = d.dv <= 64 || (d.dk > 64 && d.type == bw::Elem::kF16) ? 64 : 128;
  d.slices = (d.dv + d.slice - 1) / d.slice;
  return d;
}

bw::DeltaGates delta_gates(const DeltaIn& x) {
  return bw::DeltaGates{head_rows(x.a), head_rows(x.b), x.a_log.data_ptr(), x.dt_bias.data_ptr(), elem_of(x.a_log, "a_log"),
                        elem_of(x.dt_bias, "dt_bias")};
}

// Checks the arguments and brings them into a form that the kernels read; the scale.
double take_delta(DeltaIn& x, const std::optional<double>& scale) {
  for (const auto& [t, name] : {std::pair<const Tensor&, const char*>{x.q, "q"}, {x.k, "k"}, {x.v, "v"}, {x.a, "a"}, {x.b, "b"},
                                {x.a_log, "a_log"}, {x.dt_bias, "dt_bias"}}) {
    plain(t, name);
    TORCH_CHECK_VALUE(t.device() == x.q.device(), name, " is on ", t.device(), ", q on ", x.q.device());
  }
  TORCH_CHECK_VALUE(x.q.dim() == 4 && x.q.sizes() == x.k.sizes() && x.v.dim() == 4 && x.v.size(0) == x.q.size(0) &&
                        x.v.size(1) == x.q.size(1),
                    "q and k must be (B, T, Hk, dk), v (B, T, H, dv) with the same B and T");
  const int64_t B = x.q.size(0), T = x.q.size(1), Hk = x.q.size(2), H = x.v.size(2), dk = x.q.size(3), dv = x.v.size(3);
  TORCH_CHECK_VALUE(Hk > 0 && H > 0 && H % Hk == 0 && H / Hk <= bw::kMostGroup, "v must have 1 to ", std::to_string(bw::kMostGroup),
                    " heads for each head of q and k");
  TORCH_CHECK_VALUE(dk >= 8 && dk % 8 == 0 && dk <= bw::kMostKeyDim, "heads of q and k must have 8 to ",
                    std::to_string(bw::kMostKeyDim), " elements, a multiple of 8");
  TORCH_CHECK_VALUE(dv >= 8 && dv % 8 == 0 && dv <= 1024, "heads of v must have 8 to 1024 elements, a multiple of 8");
  for (const Tensor* t : {&x.a, &x.b})
    TORCH_CHECK_VALUE(t->dim() == 3 && t->size(0) == B && t->size(1) == T && t->size(2) == H, "a and b must be (B, T, H)");
  for (const Tensor* t : {&x.a_log, &x.dt_bias}) TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == H, "a_log and dt_bias must be (H,)");
  for (const Tensor* t : {&x.k, &x.v, &x.a, &x.b})
    TORCH_CHECK_TYPE(t->scalar_type() == x.q.scalar_type(), "q, k, v, a and b must be of one type, got ", x.q.scalar_type(), " and ",
                     t->scalar_type());
  // 2^31 - 1 blocks at most, of one value head's slice of 32 columns
  TORCH_CHECK_VALUE(T < (int64_t(1) << 31) - 64 && B * H * ((T + 63) / 64 + 1) * ((dv + 31) / 32) < (int64_t(1) << 31),
                    "the batch has too many tokens and heads for one call");
  for (Tensor* t : {&x.q, &x.k, &x.v})
    if (t->stride(3) != 1) *t = t->contiguous();
  x.a_log = x.a_log.contiguous();
  x.dt_bias = x.dt_bias.contiguous();
  if (!scale.has_value()) return 1.0 / std::sqrt((double)dk);
  TORCH_CHECK_VALUE(*scale > 0 && std::isfinite(*scale), "scale must be positive");
  return *scale;
}

Tensor take_state(const Tensor& state, const DeltaIn& x, const char* name) {
  plain(state, name);
  const std::vector<int64_t> want{x.q.size(0), x.v.size(2), x.q.size(3), x.v.size(3)};
  TORCH_CHECK_VALUE(state.device() == x.q.device() && state.sizes() == at::IntArrayRef(want), name,
                    " must be (B, H, dk, dv) on the device of q");
  TORCH_CHECK_TYPE(state.scalar_type() == torch::kFloat32, name, " must be float32, got ", state.scalar_type());
  return state;
}

// The forward's workspace, kept for the backward where there is one.
struct Kept {
  Tensor tiles, floats;  // keys, queries, solve, attend, writes, states; total, beta, rk, rq
};

// Bytes of the tiles and numbers of the floats of each part.
struct KeptSizes {
  int64_t rows, square, column, state, n, m, keys, writes, states;
  KeptSizes(const bw::DeltaDims& d, bool keep) {
    const int64_t parts = d.type == bw::Elem::kF16 ? 2 : 1, panels = d.dk <= 64 ? 1 : 2;
    rows = parts * panels * bw::kChunk * 128;  // q or k of a chunk
    square = 2 * bw::kChunk * 128;
    column = (int64_t)d.slices * d.slice * 128;  // a chunk's values, one half of them
    state = 2 * column * panels;
    n = (int64_t)d.B * d.H * d.chunks;
    m = (int64_t)d.B * d.Hk * d.chunks;
    keys = m * rows;
    writes = keep ? n * 2 * column : 0;
    states = keep ? (int64_t)d.B * d.H * d.chunks * state : 0;
  }
};

Kept make_kept(const bw::DeltaDims& d, const Tensor& like, bool keep) {
  const KeptSizes z(d, keep);
  return Kept{torch::empty({2 * z.keys + 2 * z.n * z.square + z.writes + z.states}, like.options().dtype(torch::kUInt8)),
              torch::empty({(3 * z.n + 2 * z.m) * bw::kChunk}, like.options().dtype(torch::kFloat32))};
}

bw::DeltaKept kept_parts(const bw::DeltaDims& d, const Kept& k, bool keep) {
  const KeptSizes z(d, keep);
  bw::DeltaKept p;
  p.keys = k.tiles.data_ptr<uint8_t>();
  p.queries = p.keys + z.keys;
  p.solve = p.queries + z.keys;
  p.attend = p.solve + z.n * z.square;
  p.writes = keep ? p.attend + z.n * z.square : nullptr;
  p.states = keep ? p.writes + z.writes : nullptr;
  float* f = k.floats.data_ptr<float>();
  p.total = reinterpret_cast<float2*>(f);
  p.beta = f + 2 * z.n * bw::kChunk;
  p.rk = p.beta + z.n * bw::kChunk;
  p.rq = p.rk + z.m * bw::kChunk;
  return p;
}

// {out, last state (or nothing)}; what it leaves in `kept`.
std::pair<Tensor, Tensor> delta_fwd(const DeltaIn& x, const OptTensor& first, bool want_last, double scale, const Tensor& err,
                                    bool keep, Kept& kept) {
  const c10::cuda::CUDAGuard guard(x.q.device());
  bw::DeltaFwd f;
  f.d = delta_dims(x, scale);
  f.q = head_rows(x.q);
  f.k = head_rows(x.k);
  f.v = head_rows(x.v);
  f.g = delta_gates(x);
  kept = make_kept(f.d, x.q, keep);
  f.keep = kept_parts(f.d, kept, keep);
  check_like(err, "err", torch::kInt32, x.q);
  f.err = err.data_ptr<int>();
  auto out = torch::empty({f.d.B, f.d.T, f.d.H, f.d.dv}, x.v.options());
  Tensor last;
  if (want_last) last = torch::empty({f.d.B, f.d.H, f.d.dk, f.d.dv}, x.q.options().dtype(torch::kFloat32));
  f.first = floats(first);
  f.last = want_last ? last.data_ptr<float>() : nullptr;
  f.out = out.data_ptr();
  launches += bw::delta_rule_fwd(f, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {out, last};
}

struct GatedDelta : torch::autograd::Function<GatedDelta> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& a,
                               const Tensor& b, const Tensor& a_log, const Tensor& dt_bias, const OptTensor& first, bool want_last,
                               double scale, const Tensor& err) {
    Kept kept;
    auto [out, last] = delta_fwd(DeltaIn{q, k, v, a, b, a_log, dt_bias}, first, want_last, scale, err, true, kept);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, v, a, b, a_log, dt_bias, kept.tiles, kept.floats});
    ctx->saved_data["err"] = err;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["first"] = first.has_value();
    if (!want_last) return {out};
    return {out, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list grads(11);
    const bool handed = g.size() > 1 && g[1].defined();
    if (!g[0].defined() && !handed) return grads;
    const auto s = ctx->get_saved_variables();
    const DeltaIn x{s[0], s[1], s[2], s[3], s[4], s[5], s[6]};
    const c10::cuda::CUDAGuard guard(x.q.device());
    bw::DeltaBwd w;
    w.d = delta_dims(x, ctx->saved_data["scale"].toDouble());
    w.q = head_rows(x.q);
    w.k = head_rows(x.k);
    w.v = head_rows(x.v);
    w.g = delta_gates(x);
    w.keep = kept_parts(w.d, Kept{s[7], s[8]}, true);
    const Tensor err = error_word(ctx);
    w.err = err.data_ptr<int>();
    const Tensor g_out = g[0].defined() ? g[0].contiguous() : torch::zeros({w.d.B, w.d.T, w.d.H, w.d.dv}, x.v.options());
    w.g_out = g_out.data_ptr();
    Tensor g_last;
    if (handed) g_last = g[1].contiguous();
    w.g_last = handed ? g_last.data_ptr<float>() : nullptr;
    const KeptSizes z(w.d, true);
    const int64_t parts = w.d.type == bw::Elem::kF16 ? 2 : 1;
    auto tiles = torch::empty({z.n * (z.state + (2 + parts) * z.column)}, x.q.options().dtype(torch::kUInt8));
    auto part = torch::empty({2 * z.n}, x.q.options().dtype(torch::kFloat32));
    w.dstates = tiles.data_ptr<uint8_t>();
    w.dreads = w.dstates + z.n * z.state;
    w.douts = w.dreads + z.n * 2 * z.column;
    w.part = part.data_ptr<float>();
    for (int i = 0; i < 7; ++i) grads[i] = torch::empty(s[i].sizes(), s[i].options());
    w.dq = grads[0].data_ptr();
    w.dk = grads[1].data_ptr();
    w.dv = grads[2].data_ptr();
    w.da = grads[3].data_ptr();
    w.db = grads[4].data_ptr();
    w.da_log = grads[5].data_ptr();
    w.ddt_bias = grads[6].data_ptr();
    w.dfirst = nullptr;
    if (ctx->saved_data["first"].toBool()) {
      grads[7] = torch::empty({w.d.B, w.d.H, w.d.dk, w.d.dv}, x.q.options().dtype(torch::kFloat32));
      w.dfirst = grads[7].data_ptr<float>();
    }
    launches += bw::delta_rule_bwd(w, at::cuda::getCurrentCUDAStream());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    return once(std::move(grads), "gated_delta_rule");
  }
};

std::pair<Tensor, OptTensor> gated_delta_rule(Tensor q, Tensor k, Tensor v, Tensor a, Tensor b, Tensor a_log, Tensor dt_bias,
                                              OptTensor first, bool want_last, std::optional<double> scale, Tensor err) {
  DeltaIn x{q, k, v, a, b, a_log, dt_bias};
  const double by = take_delta(x, scale);
  TORCH_CHECK_TYPE(x.q.scalar_type() == torch::kBFloat16 || x.q.scalar_type() == torch::kHalf,
                   "q, k, v, a and b must be bfloat16 or float16 on the GPU, got ", x.q.scalar_type());
  if (first.has_value()) first = take_state(*first, x, "initial_state").contiguous();
  bool tracked = first.has_value() && wants_grad(*first);
  for (const Tensor* t : {&x.q, &x.k, &x.v, &x.a, &x.b, &x.a_log, &x.dt_bias}) tracked = tracked || wants_grad(*t);
  if (!tracked) {
    Kept kept;
    auto [out, last] = delta_fwd(x, first, want_last, by, err, false, kept);
    return {out, want_last ? OptTensor(last) : std::nullopt};
  }
  auto out = GatedDelta::apply(x.q, x.k, x.v, x.a, x.b, x.a_log, x.dt_bias, first, want_last, by, err);
  return {out[0], want_last ? OptTensor(out[1]) : std::nullopt};
}

// Whether no two heads of a state, each dense in itself, share memory.
bool heads_apart(const Tensor& state) {
  const int64_t B = state.size(0), H = state.size(1), sb = state.stride(0), sh = state.stride(1), one = state.size(2) * state.size(3);
  if (state.numel() == 0 || (B == 1 && H == 1)) return true;
  if ((B > 1 && sb < one) || (H > 1 && sh < one)) return false;
  if (B == 1 || H == 1 || sb >= (H - 1) * sh + one || sh >= (B - 1) * sb + one) return true;
  for (int64_t h = 1; h < H; ++h) {  // the two sequences whose first head is nearest to head h of another one
    const int64_t b = h * sh / sb, past = h * sh - b * sb;
    if ((b < B && past < one) || (b + 1 < B && sb - past < one)) return false;
  }
  return true;
}

Tensor gated_delta_step(Tensor q, Tensor k, Tensor v, Tensor a, Tensor b, Tensor a_log, Tensor dt_bias, Tensor state,
                        std::optional<double> scale, Tensor err) {
  DeltaIn x{q, k, v, a, b, a_log, dt_bias};
  const double by = take_delta(x, scale);
  elem_of(x.q, "q, k, v, a and b");
  take_state(state, x, "state");
  for (const Tensor* t : {&x.q, &x.k, &x.v, &x.a, &x.b, &x.a_log, &x.dt_bias, &state})
    TORCH_CHECK(!wants_grad(*t), "gated_delta_step has no gradient: call it under torch.no_grad(), or gated_delta_rule");
  const int64_t dk = x.q.size(3), dv = x.v.size(3);
  TORCH_CHECK_VALUE((state.stride(3) == 1 && state.stride(2) == dv && state.stride(1) % 4 == 0 && state.stride(0) % 4 == 0 &&
                     at_multiple(state.data_ptr(), 16)) || state.numel() == 0,
                    "state must be contiguous along dk and dv, each head's on a 16-byte boundary");
  TORCH_CHECK_VALUE(heads_apart(state), "state: the heads must not overlap");
  const c10::cuda::CUDAGuard guard(x.q.device());
  bw::DeltaStep s;
  s.d = delta_dims(x, by);
  s.q = head_rows(x.q);
  s.k = head_rows(x.k);
  s.v = head_rows(x.v);
  s.g = delta_gates(x);
  auto out = torch::empty({s.d.B, s.d.T, s.d.H, s.d.dv}, x.v.options());
  s.state = state.data_ptr<float>();
  s.ssb = state.stride(0);
  s.ssh = state.stride(1);
  s.out = out.data_ptr();
  check_like(err, "err", torch::kInt32, x.q);
  s.err = err.data_ptr<int>();
  bw::delta_step(s, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  ++launches;
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  return out;
}

}  // namespace

namespace bw {

void register_trajectory(pybind11::module_& m) {
  m.def("adamw_step", &::adamw_step, "AdamW step of many tensors, moments in 32 or 8 bits");
  m.def("token_scores", &::token_scores, "log-probabilities, entropies and best alternatives from logits");
  m.def("gated_delta_rule", &::gated_delta_rule, "gated delta rule in chunks");
  m.def("gated_delta_step", &::gated_delta_step, "gated delta rule token by token, the state updated in place");
  m.def("trajectory_launches", [] { return launches.load(); }, "kernels that these functions launched");
}

}  // namespace bw
