// flash_train.torch.expert_routing over ftcuda_expert_routing and its gradient.
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>

#include <limits>
#include <optional>
#include <tuple>

#include <ftcuda/training.h>

#include "training.hpp"

namespace flash_train_torch {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

FtcudaRouting describe(const at::Tensor& logits, std::int64_t top_k, bool normalize) {
    FtcudaRouting r{};
    r.logits     = logits.data_ptr();
    r.tokens     = static_cast<std::uint64_t>(logits.size(0));
    r.row_stride = logits.stride(0);
    r.experts    = static_cast<std::uint32_t>(logits.size(1));
    r.top_k      = static_cast<std::uint32_t>(top_k);
    r.normalize  = normalize ? 1 : 0;
    r.element    = elementOf(logits);
    r.device     = logits.device().index();
    return r;
}

class ExpertRouting : public torch::autograd::Function<ExpertRouting> {
  public:
    static variable_list forward(AutogradContext* context, const at::Tensor& logits, const std::optional<at::Tensor>& mask, std::int64_t top_k, bool normalize) {
        const c10::cuda::CUDAGuard guard(logits.device());
        FtcudaRouting r            = describe(logits, top_k, normalize);
        r.mask                     = mask.has_value() ? static_cast<const std::uint8_t*>(mask->data_ptr()) : nullptr;
        const auto floats          = logits.options().dtype(at::kFloat).requires_grad(false);
        const auto integers        = floats.dtype(at::kInt);
        at::Tensor weights         = at::empty({logits.size(0), top_k}, floats);
        at::Tensor experts         = at::empty({logits.size(0), top_k}, integers);
        at::Tensor counts          = at::empty({logits.size(1)}, integers);
        at::Tensor routed          = at::empty({}, integers);
        at::Tensor loss            = at::empty({}, floats);
        const std::uint64_t bytes  = ftcuda_expert_routing_workspace_bytes(&r);
        const at::Tensor workspace = workspaceFor(bytes, logits);
        Message message;
        const int status = ftcuda_expert_routing(&r, weights.data_ptr<float>(), experts.data_ptr<std::int32_t>(), counts.data_ptr<std::int32_t>(),
                                                 routed.data_ptr<std::int32_t>(), loss.data_ptr<float>(), workspace.data_ptr(), bytes,
                                                 c10::cuda::getCurrentCUDAStream(r.device).stream(), message.text, sizeof message.text);
        TORCH_CHECK(status == 0, "flash_train expert_routing failed: ", message.text);
        context->set_materialize_grads(false);
        context->mark_non_differentiable({experts, counts, routed});
        context->save_for_backward({logits, weights, experts, counts, routed});
        context->saved_data["normalize"] = normalize;
        return {weights, experts, counts, loss, routed};
    }

    static variable_list backward(AutogradContext* context, const variable_list& gradients) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "expert_routing has no second derivative (create_graph=True)");
        const variable_list saved = context->get_saved_variables();
        const at::Tensor &logits = saved[0], &weights = saved[1], &experts = saved[2], &counts = saved[3], &routed = saved[4];
        at::Tensor grad_weights = gradients[0], grad_loss = gradients[3];
        if (!grad_weights.defined() && !grad_loss.defined()) { return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()}; }
        if (grad_weights.defined()) { grad_weights = grad_weights.to(at::kFloat).contiguous(); }
        if (grad_loss.defined()) { grad_loss = grad_loss.to(at::kFloat).contiguous(); }
        const c10::cuda::CUDAGuard guard(logits.device());
        const FtcudaRouting r  = describe(logits, weights.size(1), context->saved_data["normalize"].toBool());
        at::Tensor grad_logits = at::empty(logits.sizes(), logits.options().requires_grad(false));
        Message message;
        const int status = ftcuda_expert_routing_backward(
            &r, weights.data_ptr<float>(), experts.data_ptr<std::int32_t>(), counts.data_ptr<std::int32_t>(), routed.data_ptr<std::int32_t>(),
            grad_weights.defined() ? grad_weights.data_ptr<float>() : nullptr, grad_loss.defined() ? grad_loss.data_ptr<float>() : nullptr,
            grad_logits.data_ptr(), grad_logits.stride(0), c10::cuda::getCurrentCUDAStream(r.device).stream(), message.text, sizeof message.text);
        TORCH_CHECK(status == 0, "flash_train expert_routing's gradient failed: ", message.text);
        return {grad_logits, at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> expertRouting(const at::Tensor& logits, std::int64_t top_k, bool normalize,
                                                                         const std::optional<at::Tensor>& mask) {
    TORCH_CHECK(logits.is_cuda() && logits.layout() == at::kStrided, "logits must be a dense device tensor");
    TORCH_CHECK(elementOf(logits) != 0, "logits must be FP32, FP16 or BF16");
    TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) >= 1 && logits.size(-1) <= 1024, "logits must have 1 to 1024 experts along the last dimension");
    TORCH_CHECK(top_k >= 1 && top_k <= logits.size(-1) && top_k <= 32, "top_k must be from 1 to the number of experts, and at most 32");
    TORCH_CHECK(!logits.is_neg(), "logits must not be a negated view");
    const std::int64_t experts = logits.size(-1);
    const at::Tensor flat      = logits.dim() == 2 ? logits : logits.reshape({logits.numel() / experts, experts});
    TORCH_CHECK(flat.stride(1) == 1 || experts == 1, "the experts of a token must be neighbours in memory");
    std::optional<at::Tensor> bytes;
    if (mask.has_value()) {
        TORCH_CHECK(mask->scalar_type() == at::kBool && mask->device() == logits.device(), "mask must be a tensor of truth values on the logits' device");
        TORCH_CHECK(mask->sizes() == logits.sizes().slice(0, logits.dim() - 1), "mask must have a value for each token");
        bytes = mask->contiguous();
    }
    const variable_list out = ExpertRouting::apply(flat, bytes, top_k, normalize);
    if (logits.dim() == 2) { return {out[0], out[1], out[2], out[3]}; }
    std::vector<std::int64_t> shape(logits.sizes().begin(), logits.sizes().end());
    shape.back() = top_k;
    return {out[0].view(shape), out[1].view(shape), out[2], out[3]};
}

}  // namespace

void registerExpertRouting(pybind11::module_& module) {
    module.def("_expert_routing", &expertRouting, pybind11::arg("logits"), pybind11::arg("top_k"), pybind11::arg("normalize"), pybind11::arg("mask"));
}

}  // namespace flash_train_torch
