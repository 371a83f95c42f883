// PyTorch-facing host code of the operators around the experts: argument checks and output allocation of
// the expert selection and of the distillation loss.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <vector>

#include "kernels.h"
#include "torch_ops.h"

namespace mb {

namespace {

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

DType float_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return kF32;
    case at::kHalf: return kF16;
    case at::kBFloat16: return kBF16;
    default: TORCH_CHECK(false, "expected float32 / float16 / bfloat16, got ", t);
  }
}

SelectArgs select_args(const at::Tensor& logits, int64_t top_k, bool use_sigmoid, int64_t groups, int64_t top_groups,
                       int64_t norm_p, double scale) {
  TORCH_CHECK(logits.is_cuda() && logits.is_contiguous() && logits.dim() == 2,
              "select_experts expects contiguous CUDA logits[tokens, experts]");
  const int64_t experts = logits.size(1);
  TORCH_CHECK(experts >= 1 && experts <= kRouterMaxExperts && top_k >= 1 && top_k <= kSelectMaxTopK,
              "select_experts takes up to 1024 experts and top_k up to 32");
  TORCH_CHECK(groups >= 1 && groups <= kSelectMaxGroups && experts % groups == 0 && top_groups >= 1 &&
                  top_groups <= groups && top_k <= top_groups * (experts / groups),
              "select_experts: groups must divide the experts, and top_groups of them hold top_k");
  TORCH_CHECK(norm_p >= 0 && norm_p <= 2, "select_experts: norm_p is 0, 1 or 2");
  SelectArgs a{};
  a.tokens = logits.size(0);
  a.experts = int(experts);
  a.top_k = int(top_k);
  a.groups = int(groups);
  a.top_groups = int(top_groups);
  a.norm_p = int(norm_p);
  a.use_sigmoid = use_sigmoid;
  a.scale = float(scale);
  TORCH_CHECK(a.tokens <= (int64_t(1) << 32), "select_experts: too many tokens");
  return a;
}

}  // namespace

std::vector<at::Tensor> select_experts_forward(const at::Tensor& logits, int64_t top_k, bool use_sigmoid,
                                               const OptTensor& bias, int64_t groups, int64_t top_groups,
                                               int64_t norm_p, double scale) {
  SelectArgs a = select_args(logits, top_k, use_sigmoid, groups, top_groups, norm_p, scale);
  if (bias.has_value()) {
    TORCH_CHECK(bias->device() == logits.device() && bias->is_contiguous() && bias->scalar_type() == at::kFloat &&
                    bias->dim() == 1 && bias->size(0) == a.experts,
                "select_experts: bias must be a contiguous float32 vector of the experts on the logits' device");
    a.bias = bias->data_ptr<float>();
  }
  const DType code = float_code(logits.scalar_type());
  c10::cuda::CUDAGuard guard(logits.device());
  at::Tensor scores = at::empty_like(logits);
  at::Tensor weights = at::empty({a.tokens, top_k}, logits.options());
  at::Tensor ids = at::empty({a.tokens, top_k}, logits.options().dtype(at::kLong));
  if (a.tokens == 0) return {scores, weights, ids};
  C10_CUDA_CHECK(select_experts_fwd(code, logits.data_ptr(), a, scores.data_ptr(), weights.data_ptr(),
                                    ids.data_ptr<int64_t>(), stream()));
  count_launches(1);
  return {scores, weights, ids};
}

at::Tensor select_experts_backward(const at::Tensor& logits, const at::Tensor& experts, const OptTensor& dscores,
                                   const OptTensor& dweights, bool use_sigmoid, int64_t norm_p, double scale) {
  TORCH_CHECK(experts.dim() == 2 && experts.is_contiguous() && experts.device() == logits.device() &&
                  experts.scalar_type() == at::kLong && logits.dim() == 2 && experts.size(0) == logits.size(0),
              "select_experts: experts must be the forward pass's ids");
  const SelectArgs a = select_args(logits, experts.size(1), use_sigmoid, 1, 1, norm_p, scale);
  int64_t stride = 0;
  if (dscores.has_value()) {
    TORCH_CHECK(dscores->device() == logits.device() && dscores->sizes() == logits.sizes() &&
                    dscores->scalar_type() == logits.scalar_type() &&
                    (a.experts == 1 || dscores->stride(1) == 1 || a.tokens == 0),
                "select_experts: the scores' gradient must be like the logits, with unit stride in the experts");
    stride = dscores->stride(0);
    TORCH_CHECK(a.tokens <= 1 || stride == 0 || stride == a.experts,
                "select_experts: the scores' gradient has one row for all tokens or dense rows");
  }
  if (dweights.has_value())
    TORCH_CHECK(dweights->device() == logits.device() && dweights->sizes() == experts.sizes() &&
                    dweights->is_contiguous() && dweights->scalar_type() == logits.scalar_type(),
                "select_experts: the weights' gradient must be contiguous and like the weights");
  c10::cuda::CUDAGuard guard(logits.device());
  at::Tensor dlogits = at::empty_like(logits);
  if (a.tokens == 0) return dlogits;
  C10_CUDA_CHECK(select_experts_bwd(float_code(logits.scalar_type()), logits.data_ptr(), a, experts.data_ptr<int64_t>(),
                                    dscores.has_value() ? dscores->data_ptr() : nullptr, stride,
                                    dweights.has_value() ? dweights->data_ptr() : nullptr, dlogits.data_ptr(),
                                    stream()));
  count_launches(1);
  return dlogits;
}

namespace {

DistillArgs distill_args(const at::Tensor& logits, const at::Tensor& values, const at::Tensor& ids,
                         const OptTensor& targets, double temperature, double hard_weight, double scale) {
  TORCH_CHECK(logits.is_cuda() && logits.is_contiguous() && logits.dim() == 2 && logits.size(1) >= 1 &&
                  logits.size(1) < (int64_t(1) << 31) && logits.size(0) < (int64_t(1) << 31),
              "distillation expects contiguous CUDA logits[rows, vocab]");
  TORCH_CHECK(values.dim() == 2 && values.size(0) == logits.size(0) && values.sizes() == ids.sizes() &&
                  values.is_contiguous() && ids.is_contiguous() && values.device() == logits.device() &&
                  ids.device() == logits.device() && values.size(1) >= 1 && values.size(1) <= kDistillMaxTop,
              "distillation expects the teacher's logits and their ids as contiguous [rows, top], top up to 1024");
  TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt,
              "distillation: the teacher's ids are int64 or int32");
  if (targets.has_value())
    TORCH_CHECK(targets->device() == logits.device() && targets->is_contiguous() && targets->dim() == 1 &&
                    targets->size(0) == logits.size(0) && targets->scalar_type() == at::kLong,
                "distillation: targets are int64 [rows]");
  TORCH_CHECK(temperature > 0, "distillation: the temperature must be positive");
  DistillArgs a{};
  a.logits = logits.data_ptr();
  a.rows = logits.size(0);
  a.vocab = int(logits.size(1));
  a.top = int(values.size(1));
  a.values = values.data_ptr();
  a.value_type = float_code(values.scalar_type());
  a.ids = ids.data_ptr();
  a.ids64 = ids.scalar_type() == at::kLong;
  a.targets = targets.has_value() ? targets->data_ptr<int64_t>() : nullptr;
  a.temperature = float(temperature);
  a.hard_weight = float(hard_weight);
  a.scale = float(scale);
  return a;
}

}  // namespace

// {loss[rows], stats[rows, 3], gradient of scale * sum(loss) (undefined unless wanted; the logits themselves
// when `in_place`)}.
std::vector<at::Tensor> distill_forward(const at::Tensor& logits, const at::Tensor& values, const at::Tensor& ids,
                                        const OptTensor& targets, double temperature, double hard_weight, double scale,
                                        bool want_grad, bool in_place) {
  DistillArgs a = distill_args(logits, values, ids, targets, temperature, hard_weight, scale);
  const DType code = float_code(logits.scalar_type());
  c10::cuda::CUDAGuard guard(logits.device());
  const auto fopts = logits.options().dtype(at::kFloat);
  at::Tensor loss = at::empty({a.rows}, fopts), stats = at::empty({a.rows, 3}, fopts), grad;
  if (want_grad) grad = in_place ? logits : at::empty_like(logits);
  if (a.rows == 0) return {loss, stats, grad};
  a.status = device_status(logits.device());
  C10_CUDA_CHECK(distill_fwd(code, a, loss.data_ptr<float>(), stats.data_ptr<float>(),
                             want_grad ? grad.data_ptr() : nullptr, stream()));
  count_launches(1);
  return {loss, stats, grad};
}

at::Tensor distill_backward(const at::Tensor& logits, const at::Tensor& values, const at::Tensor& ids,
                            const OptTensor& targets, const at::Tensor& stats, const at::Tensor& grad_out,
                            double temperature, double hard_weight, double scale) {
  const DistillArgs a = distill_args(logits, values, ids, targets, temperature, hard_weight, scale);
  TORCH_CHECK(stats.device() == logits.device() && stats.is_contiguous() && stats.numel() == 3 * a.rows &&
                  grad_out.device() == logits.device() && grad_out.scalar_type() == at::kFloat &&
                  grad_out.numel() == 1,
              "distillation: the backward pass takes the forward pass's statistics and a float32 scalar");
  c10::cuda::CUDAGuard guard(logits.device());
  at::Tensor grad = at::empty_like(logits);
  if (a.rows == 0) return grad;
  C10_CUDA_CHECK(distill_bwd(float_code(logits.scalar_type()), a, stats.data_ptr<float>(), grad_out.data_ptr<float>(),
                             grad.data_ptr(), stream()));
  count_launches(1);
  return grad;
}

void scale_unless_one_op(at::Tensor x, const at::Tensor& factor) {
  TORCH_CHECK(x.is_cuda() && x.is_contiguous() && factor.device() == x.device() && factor.numel() == 1 &&
                  factor.scalar_type() == at::kFloat && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0,
              "scale_unless_one_ expects a contiguous CUDA tensor and a float32 scalar");
  c10::cuda::CUDAGuard guard(x.device());
  if (x.numel() == 0) return;
  C10_CUDA_CHECK(scale_unless_one(float_code(x.scalar_type()), x.data_ptr(), x.numel(), factor.data_ptr<float>(),
                                  at::cuda::getCurrentDeviceProperties()->multiProcessorCount, stream()));
  count_launches(1);
}

}  // namespace mb
