// PyTorch-facing host code of the operators around the experts: argument checks and output allocation of
// the expert selection and of the distillation loss.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "kernels.h"
#include "torch_ops.h"

namespace mb {

namespace {

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }
int sm_count() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

DType float_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return kF32;
    case at::kHalf: return kF16;
    case at::kBFloat16: return kBF16;
    default: TORCH_CHECK(false, "expected float32 / float16 / bfloat16, got ", t);
  }
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

SelectArgs select_args(const at::Tensor& logits, int64_t top_k, bool use_sigmoid, int64_t groups, int64_t top_groups,
                       int64_t norm_p, double scale) {
  TORCH_CHECK_VALUE(logits.is_cuda() && logits.dim() == 2 && logits.size(0) <= (int64_t(1) << 32),
                    "select_experts expects CUDA logits[tokens, experts]");
  const int64_t experts = logits.size(1);
  TORCH_CHECK_VALUE(experts >= 1 && experts <= kRouterMaxExperts, "select_experts takes 1 to ", kRouterMaxExperts,
                    " experts, got ", experts);
  TORCH_CHECK_VALUE(groups >= 1 && groups <= kSelectMaxGroups && experts % groups == 0, "groups must divide the ", experts,
                    " experts and be at most ", kSelectMaxGroups, ", got ", groups);
  TORCH_CHECK_VALUE(top_groups >= 1 && top_groups <= groups, "top_groups must lie in [1, ", groups, "], got ", top_groups);
  TORCH_CHECK_VALUE(top_k >= 1 && top_k <= kSelectMaxTopK && top_k <= top_groups * (experts / groups),
                    "top_k must be at least 1, at most ", kSelectMaxTopK, ", and no more than the chosen groups hold, got ",
                    top_k);
  TORCH_CHECK_VALUE(norm_p >= 0 && norm_p <= 2, "norm_p must be None, 1 or 2");
  SelectArgs a{};
  a.tokens = logits.size(0);
  a.experts = int(experts);
  a.top_k = int(top_k);
  a.groups = int(groups);
  a.top_groups = int(top_groups);
  a.norm_p = int(norm_p);
  a.use_sigmoid = use_sigmoid;
  a.scale = float(scale);
  return a;
}

std::vector<at::Tensor> select_forward(const at::Tensor& logits, SelectArgs a, const OptTensor& bias) {
  if (bias.has_value()) {
    TORCH_CHECK_VALUE(bias->device() == logits.device() && bias->is_contiguous() && bias->scalar_type() == at::kFloat &&
                          bias->dim() == 1 && bias->size(0) == a.experts,
                      "bias must be a dense float32 vector with one entry per expert, on the device of the logits");
    a.bias = bias->data_ptr<float>();
  }
  const DType code = float_code(logits.scalar_type());
  c10::cuda::CUDAGuard guard(logits.device());
  at::Tensor scores = at::empty_like(logits);
  at::Tensor weights = at::empty({a.tokens, a.top_k}, logits.options());
  at::Tensor ids = at::empty({a.tokens, a.top_k}, logits.options().dtype(at::kLong));
  if (a.tokens == 0) return {scores, weights, ids};
  C10_CUDA_CHECK(select_experts_fwd(code, logits.data_ptr(), a, scores.data_ptr(), weights.data_ptr(),
                                    ids.data_ptr<int64_t>(), stream()));
  count_launches(1);
  return {scores, weights, ids};
}

at::Tensor select_backward(const at::Tensor& logits, const SelectArgs& a, const at::Tensor& ids, at::Tensor dscores,
                           at::Tensor dweights) {
  int64_t stride = 0;
  if (dscores.defined()) {
    // One row that is expanded over the tokens is read as it is.
    if (!(dscores.stride(1) == 1 && (dscores.stride(0) == 0 || dscores.stride(0) == a.experts))) dscores = dscores.contiguous();
    stride = a.tokens > 1 ? dscores.stride(0) : 0;
  }
  if (dweights.defined()) dweights = dweights.contiguous();
  c10::cuda::CUDAGuard guard(logits.device());
  at::Tensor dlogits = at::empty_like(logits);
  if (a.tokens == 0) return dlogits;
  C10_CUDA_CHECK(select_experts_bwd(float_code(logits.scalar_type()), logits.data_ptr(), a, ids.data_ptr<int64_t>(),
                                    dscores.defined() ? dscores.data_ptr() : nullptr, stride,
                                    dweights.defined() ? dweights.data_ptr() : nullptr, dlogits.data_ptr(), stream()));
  count_launches(1);
  return dlogits;
}

// A C++ node: the host passes it in a few microseconds each way, a Python one in some 20, which is more than
// the kernels of all but the largest calls take.
struct Select : torch::autograd::Function<Select> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, int64_t top_k, bool use_sigmoid,
                               const OptTensor& bias, int64_t groups, int64_t top_groups, int64_t norm_p, double scale) {
    auto out = select_forward(logits, select_args(logits, top_k, use_sigmoid, groups, top_groups, norm_p, scale), bias);
    ctx->save_for_backward({logits, out[2]});
    ctx->saved_data["how"] = std::vector<int64_t>{use_sigmoid, norm_p};
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({out[2]});
    ctx->set_materialize_grads(false);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(8);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const auto how = ctx->saved_data["how"].toIntVector();
    const SelectArgs a = select_args(saved[0], saved[1].size(1), how[0] != 0, 1, 1, how[1],
                                     ctx->saved_data["scale"].toDouble());
    out[0] = select_backward(saved[0], a, saved[1], grads[0], grads[1]);
    return once_differentiable(out, "select_experts");
  }
};

}  // namespace

// {scores[tokens, experts], weights[tokens, top_k], ids[tokens, top_k]}, differentiable in the logits.
std::vector<at::Tensor> select_experts(const at::Tensor& logits, int64_t top_k, bool use_sigmoid, const OptTensor& bias,
                                       int64_t groups, int64_t top_groups, int64_t norm_p, double scale) {
  const at::Tensor dense = logits.contiguous();
  const OptTensor fixed = bias.has_value() ? OptTensor(bias->detach().contiguous()) : OptTensor();
  if (at::GradMode::is_enabled() && dense.requires_grad())
    return Select::apply(dense, top_k, use_sigmoid, fixed, groups, top_groups, norm_p, scale);
  return select_forward(dense, select_args(dense, top_k, use_sigmoid, groups, top_groups, norm_p, scale), fixed);
}

namespace {

DistillArgs distill_args(const at::Tensor& logits, const at::Tensor& values, const at::Tensor& ids,
                         const OptTensor& targets, double temperature, double hard_weight) {
  TORCH_CHECK_VALUE(logits.is_cuda() && logits.is_contiguous() && logits.dim() == 2 && logits.size(1) >= 1 &&
                        logits.size(1) < (int64_t(1) << 31) && logits.size(0) < (int64_t(1) << 31),
                    "distillation expects logits[rows, vocab]");
  TORCH_CHECK_VALUE(values.dim() == 2 && values.size(0) == logits.size(0) && values.sizes() == ids.sizes(),
                    "distillation expects the teacher's logits and ids as [rows, top], one row per row of logits");
  TORCH_CHECK_VALUE(values.size(1) >= 1 && values.size(1) <= kDistillMaxTop, "distillation takes 1 to ", kDistillMaxTop,
                    " teacher logits a row");
  TORCH_CHECK_VALUE(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt,
                    "the teacher's ids must be int32 or int64");
  TORCH_CHECK_VALUE(values.is_floating_point(), "the teacher's logits must be floating-point");
  TORCH_CHECK_VALUE(std::isfinite(temperature) && temperature > 0, "the temperature must be positive, got ", temperature);
  TORCH_CHECK_VALUE(std::isfinite(hard_weight) && hard_weight >= 0, "hard_weight must not be negative, got ", hard_weight);
  TORCH_CHECK_VALUE(hard_weight == 0 || targets.has_value(), "hard_weight needs targets");
  TORCH_CHECK_VALUE(values.device() == logits.device() && ids.device() == logits.device() &&
                        (!targets.has_value() || targets->device() == logits.device()),
                    "the teacher's logits, its ids and the targets must be on the device of the logits");
  if (targets.has_value())
    TORCH_CHECK_VALUE(targets->dim() == 1 && targets->size(0) == logits.size(0) && targets->scalar_type() == at::kLong,
                      "targets must be int64 with one entry per row");
  DistillArgs a{};
  a.logits = logits.data_ptr();
  a.rows = logits.size(0);
  a.vocab = int(logits.size(1));
  a.top = int(values.size(1));
  a.values = values.data_ptr();
  a.value_type = float_code(values.scalar_type());
  a.ids = ids.data_ptr();
  a.ids64 = ids.scalar_type() == at::kLong;
  a.targets = targets.has_value() && hard_weight != 0 ? targets->data_ptr<int64_t>() : nullptr;
  a.temperature = float(temperature);
  a.hard_weight = float(hard_weight);
  a.scale = 1.f / float(std::max<int64_t>(a.rows, 1));
  return a;
}

struct Distilled {
  at::Tensor loss, stats, grad;        // mean loss, row statistics, its gradient (undefined unless wanted)
};

Distilled distill_forward(const at::Tensor& logits, const at::Tensor& values, const at::Tensor& ids,
                          const OptTensor& targets, double temperature, double hard_weight, bool want_grad,
                          bool in_place) {
  DistillArgs a = distill_args(logits, values, ids, targets, temperature, hard_weight);
  const DType code = float_code(logits.scalar_type());
  c10::cuda::CUDAGuard guard(logits.device());
  const auto fopts = logits.options().dtype(at::kFloat);
  Distilled d;
  if (want_grad) d.grad = in_place ? logits : at::empty_like(logits);
  if (a.rows == 0) {
    d.loss = at::zeros({}, fopts);
    d.stats = at::empty({0, 4}, fopts);
    return d;
  }
  d.loss = at::empty({}, fopts);
  d.stats = at::empty({a.rows, 4}, fopts);        // loss, maximum, sums
  a.status = device_status(logits.device());
  C10_CUDA_CHECK(distill_fwd(code, a, d.stats.data_ptr<float>(), want_grad ? d.grad.data_ptr() : nullptr, sm_count(),
                             stream()));
  C10_CUDA_CHECK(distill_mean(d.stats.data_ptr<float>(), a.rows, d.loss.data_ptr<float>(), stream()));
  count_launches(2);
  return d;
}

// The forward pass takes the gradient of the loss while it has the row, into a tensor of its own; the backward
// pass multiplies it by the incoming scalar where that is not one.  fp16 logits take it in the backward pass
// instead: unscaled it underflows, and the loss scale is only known there.
struct Distill : torch::autograd::Function<Distill> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& values,
                            const at::Tensor& ids, const OptTensor& targets, double temperature, double hard_weight) {
    Distilled d = distill_forward(logits, values, ids, targets, temperature, hard_weight,
                                  logits.scalar_type() != at::kHalf, false);
    ctx->save_for_backward({logits, values, ids, targets.has_value() ? *targets : at::Tensor(), d.stats});
    ctx->saved_data["how"] = std::vector<double>{temperature, hard_weight};
    if (d.grad.defined()) ctx->saved_data["grad"] = d.grad;
    return d.loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(6);
    const at::Tensor scale = grads[0].detach().to(at::kFloat).reshape(1);
    const auto kept = ctx->saved_data.find("grad");
    if (kept != ctx->saved_data.end()) {          // a second backward pass takes it again from the logits
      out[0] = kept->second.toTensor();
      ctx->saved_data.erase(kept);
      c10::cuda::CUDAGuard guard(out[0].device());
      C10_CUDA_CHECK(scale_unless_one(float_code(out[0].scalar_type()), out[0].data_ptr(), out[0].numel(),
                                      scale.data_ptr<float>(), sm_count(), stream()));
      count_launches(1);
      return once_differentiable(out, "distillation_loss");
    }
    const auto saved = ctx->get_saved_variables();
    const auto how = ctx->saved_data["how"].toDoubleVector();
    const OptTensor targets = saved[3].defined() ? OptTensor(saved[3]) : OptTensor();
    const DistillArgs a = distill_args(saved[0], saved[1], saved[2], targets, how[0], how[1]);
    c10::cuda::CUDAGuard guard(saved[0].device());
    out[0] = at::empty_like(saved[0]);
    if (a.rows == 0) return out;
    C10_CUDA_CHECK(distill_bwd(float_code(saved[0].scalar_type()), a, saved[4].data_ptr<float>(),
                               scale.data_ptr<float>(), out[0].data_ptr(), stream()));
    count_launches(1);
    return once_differentiable(out, "distillation_loss");
  }
};

OptTensor dense(const OptTensor& t) { return t.has_value() ? OptTensor(t->contiguous()) : t; }

}  // namespace

// Mean loss of logits[rows, vocab], differentiable in them.
at::Tensor distillation_loss(const at::Tensor& logits, const at::Tensor& values, const at::Tensor& ids,
                             const OptTensor& targets, double temperature, double hard_weight) {
  const at::Tensor z = logits.contiguous(), v = values.detach().contiguous(), i = ids.contiguous();
  if (at::GradMode::is_enabled() && z.requires_grad())
    return Distill::apply(z, v, i, dense(targets), temperature, hard_weight);
  return distill_forward(z, v, i, dense(targets), temperature, hard_weight, false, false).loss;
}

// Mean loss, and its gradient written over the logits.
std::vector<at::Tensor> distill_in_place(const at::Tensor& logits, const at::Tensor& values, const at::Tensor& ids,
                                         const OptTensor& targets, double temperature, double hard_weight) {
  Distilled d = distill_forward(logits, values.detach().contiguous(), ids.contiguous(), dense(targets), temperature,
                                hard_weight, true, true);
  return {d.loss, d.grad};
}

}  // namespace mb
