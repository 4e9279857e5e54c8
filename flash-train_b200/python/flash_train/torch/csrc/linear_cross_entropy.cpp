// flash_train.torch.linear_cross_entropy over ftcuda_linear_cross_entropy and its gradients.
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>

#include <string>

#include <ftcuda/training.h>

#include "training.hpp"

namespace flash_train_torch {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

FtcudaLinearCrossEntropy describe(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& target, std::int64_t ignore_index, std::int64_t reduction) {
    FtcudaLinearCrossEntropy q{};
    q.hidden            = hidden.data_ptr();
    q.weight            = weight.data_ptr();
    q.target            = target.data_ptr<std::int64_t>();
    q.tokens            = static_cast<std::uint64_t>(hidden.size(0));
    q.vocabulary        = static_cast<std::uint64_t>(weight.size(0));
    q.depth             = static_cast<std::uint64_t>(hidden.size(1));
    q.hidden_row_stride = hidden.stride(0);
    q.weight_row_stride = weight.stride(0);
    q.ignore_index      = ignore_index;
    q.element           = elementOf(hidden);
    q.reduction         = static_cast<std::int32_t>(reduction);
    q.device            = hidden.device().index();
    return q;
}

at::Tensor workspaceOf(const FtcudaLinearCrossEntropy& q, bool backward, const at::Tensor& like, std::uint64_t& bytes) {
    Message message;
    const int status = ftcuda_linear_cross_entropy_workspace_bytes(&q, backward ? 1 : 0, &bytes, message.text, sizeof message.text);
    TORCH_CHECK(status == 0, "flash_train linear_cross_entropy failed: ", message.text);
    return workspaceFor(bytes, like);
}

cudaStream_t streamOf(const FtcudaLinearCrossEntropy& q) { return c10::cuda::getCurrentCUDAStream(q.device).stream(); }

void* addressOf(const at::Tensor& tensor) { return tensor.defined() ? tensor.data_ptr() : nullptr; }

// The loss now, the gradients when they are asked for: the logits are computed twice.
class LinearCrossEntropy : public torch::autograd::Function<LinearCrossEntropy> {
  public:
    static at::Tensor forward(AutogradContext* context, const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& target, std::int64_t ignore_index,
                              std::int64_t reduction) {
        const c10::cuda::CUDAGuard guard(hidden.device());
        const FtcudaLinearCrossEntropy q = describe(hidden, weight, target, ignore_index, reduction);
        const auto floats                = hidden.options().dtype(at::kFloat).requires_grad(false);
        at::Tensor loss                  = reduction == FTCUDA_REDUCTION_NONE ? at::empty({hidden.size(0)}, floats) : at::empty({}, floats);
        at::Tensor lse                   = at::empty({hidden.size(0)}, floats);
        std::uint64_t bytes              = 0;
        const at::Tensor workspace       = workspaceOf(q, false, hidden, bytes);
        Message message;
        const int status = ftcuda_linear_cross_entropy(&q, loss.data_ptr<float>(), lse.data_ptr<float>(), workspace.data_ptr(), bytes, streamOf(q), message.text,
                                                       sizeof message.text);
        TORCH_CHECK(status == 0, "flash_train linear_cross_entropy failed: ", message.text);
        context->save_for_backward({hidden, weight, target, lse});
        context->saved_data["ignore_index"] = ignore_index;
        context->saved_data["reduction"]    = reduction;
        return loss;
    }

    static variable_list backward(AutogradContext* context, const variable_list& gradients) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "linear_cross_entropy has no second derivative (create_graph=True)");
        const variable_list saved = context->get_saved_variables();
        const at::Tensor &hidden = saved[0], &weight = saved[1], &target = saved[2], &lse = saved[3];
        const at::Tensor grad_loss = gradients[0].to(at::kFloat).contiguous();
        const c10::cuda::CUDAGuard guard(hidden.device());
        const FtcudaLinearCrossEntropy q =
            describe(hidden, weight, target, context->saved_data["ignore_index"].toInt(), context->saved_data["reduction"].toInt());
        at::Tensor grad_hidden, grad_weight;
        if (context->needs_input_grad(0)) { grad_hidden = at::empty(hidden.sizes(), hidden.options().requires_grad(false)); }
        if (context->needs_input_grad(1)) { grad_weight = at::empty(weight.sizes(), weight.options().requires_grad(false)); }
        std::uint64_t bytes        = 0;
        const at::Tensor workspace = workspaceOf(q, true, hidden, bytes);
        Message message;
        const int status = ftcuda_linear_cross_entropy_backward(&q, lse.data_ptr<float>(), grad_loss.data_ptr<float>(), addressOf(grad_hidden), hidden.size(1),
                                                                addressOf(grad_weight), hidden.size(1), workspace.data_ptr(), bytes, streamOf(q), message.text,
                                                                sizeof message.text);
        TORCH_CHECK(status == 0, "flash_train linear_cross_entropy's gradient failed: ", message.text);
        return {grad_hidden, grad_weight, at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

// The logits are computed once: the forward pass leaves what the gradients are made of in a tensor that the graph keeps until the backward pass. (The weight is the graph's too, and may
// come back from a saved-tensor hook as another copy; only the kept tensor's size has to stay.)
class LinearCrossEntropyStep : public torch::autograd::Function<LinearCrossEntropyStep> {
  public:
    static at::Tensor forward(AutogradContext* context, const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& target, std::int64_t ignore_index,
                              std::int64_t reduction, std::int64_t kept_bytes, std::int64_t workspace_bytes) {
        const c10::cuda::CUDAGuard guard(hidden.device());
        const FtcudaLinearCrossEntropy q = describe(hidden, weight, target, ignore_index, reduction);
        at::Tensor loss                  = at::empty({}, hidden.options().dtype(at::kFloat).requires_grad(false));
        const at::Tensor kept            = workspaceFor(static_cast<std::uint64_t>(kept_bytes), hidden);
        const at::Tensor workspace       = workspaceFor(static_cast<std::uint64_t>(workspace_bytes), hidden);
        Message message;
        const int status = ftcuda_linear_cross_entropy_step_loss_kept(&q, loss.data_ptr<float>(), kept.data_ptr(), static_cast<std::uint64_t>(kept_bytes), workspace.data_ptr(),
                                                                      static_cast<std::uint64_t>(workspace_bytes), streamOf(q), message.text, sizeof message.text);
        TORCH_CHECK(status == 0, "flash_train linear_cross_entropy failed: ", message.text);
        context->save_for_backward({hidden, weight, target, kept});
        context->saved_data["ignore_index"] = ignore_index;
        context->saved_data["reduction"]    = reduction;
        return loss;
    }

    static variable_list backward(AutogradContext* context, const variable_list& gradients) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "linear_cross_entropy has no second derivative (create_graph=True)");
        const variable_list saved = context->get_saved_variables();
        const at::Tensor &hidden = saved[0], &weight = saved[1], &target = saved[2], &kept = saved[3];
        const at::Tensor grad_loss = gradients[0].to(at::kFloat).contiguous();
        const c10::cuda::CUDAGuard guard(hidden.device());
        const FtcudaLinearCrossEntropy q =
            describe(hidden, weight, target, context->saved_data["ignore_index"].toInt(), context->saved_data["reduction"].toInt());
        variable_list out(7);
        if (context->needs_input_grad(0)) { out[0] = at::empty(hidden.sizes(), hidden.options().requires_grad(false)); }
        if (context->needs_input_grad(1)) { out[1] = at::empty(weight.sizes(), weight.options().requires_grad(false)); }
        const std::uint64_t kept_bytes = static_cast<std::uint64_t>(kept.numel());
        std::uint64_t bytes            = 0;
        Message message;
        int status = ftcuda_linear_cross_entropy_step_gradients_bytes(&q, kept_bytes, &bytes, message.text, sizeof message.text);
        TORCH_CHECK(status == 0, "flash_train linear_cross_entropy's gradient failed: ", message.text);
        const at::Tensor workspace = workspaceFor(bytes, hidden);
        status = ftcuda_linear_cross_entropy_step_gradients_kept(&q, grad_loss.data_ptr<float>(), addressOf(out[0]), hidden.size(1), addressOf(out[1]), hidden.size(1), kept.data_ptr(),
                                                                 kept_bytes, workspace.data_ptr(), bytes, streamOf(q), message.text, sizeof message.text);
        TORCH_CHECK(status == 0, "flash_train linear_cross_entropy's gradient failed: ", message.text);
        return out;
    }
};

// What the step form could not be given on a device.
RefusedWorkspace& refusedStep(std::size_t device) {
    static thread_local std::vector<RefusedWorkspace> refused;
    return ofDevice(refused, device);
}

at::Tensor linearCrossEntropy(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& target, std::int64_t ignore_index, const std::string& reduction,
                              bool recompute) {
    for (const at::Tensor* operand : {&hidden, &weight}) {
        TORCH_CHECK(operand->is_cuda() && operand->layout() == at::kStrided && !operand->is_neg(), "hidden and weight must be dense device tensors");
        TORCH_CHECK(elementOf(*operand) != 0, "hidden and weight must be FP32, FP16 or BF16");
    }
    TORCH_CHECK(hidden.scalar_type() == weight.scalar_type(), "hidden and weight must have one type");
    TORCH_CHECK(weight.dim() == 2 && hidden.dim() >= 1, "weight must be rank two, hidden rank one or more");
    TORCH_CHECK(hidden.size(-1) == weight.size(1), "hidden's last dimension must equal weight's columns");
    TORCH_CHECK(hidden.size(-1) >= 1 && weight.size(0) >= 1, "weight must not be empty");
    TORCH_CHECK(target.is_cuda() && target.scalar_type() == at::kLong, "target must be an INT64 device tensor");
    TORCH_CHECK(target.sizes() == hidden.sizes().slice(0, hidden.dim() - 1), "target must have a value for each hidden state");
    TORCH_CHECK(weight.device() == hidden.device() && target.device() == hidden.device(), "hidden, weight and target must be on the same device");
    const std::int64_t depth = hidden.size(-1);
    const std::int64_t kind  = reduction == "none" ? FTCUDA_REDUCTION_NONE : reduction == "mean" ? FTCUDA_REDUCTION_MEAN : FTCUDA_REDUCTION_SUM;
    TORCH_CHECK(kind != FTCUDA_REDUCTION_SUM || reduction == "sum", "reduction must be 'none', 'mean' or 'sum'");
    const at::Tensor flat = hidden.dim() == 2 ? hidden : hidden.reshape({hidden.numel() / depth, depth});
    TORCH_CHECK((flat.stride(1) == 1 && weight.stride(1) == 1) || depth == 1, "hidden and weight must be contiguous along their last dimension");
    const at::Tensor indices = target.reshape({-1}).contiguous();
    if (!recompute && at::GradMode::is_enabled() && (flat.requires_grad() || weight.requires_grad())) {
        const FtcudaLinearCrossEntropy q = describe(flat, weight, indices, ignore_index, kind);
        std::uint64_t kept = 0, bytes = 0;
        if (ftcuda_linear_cross_entropy_step_loss_bytes(&q, &kept, &bytes, nullptr, 0) == 0) {
            // Where the allocator has no room for all logits' exponentials, the form that goes through the vocabulary piece by piece takes less.
            RefusedWorkspace& refused = refusedStep(static_cast<std::size_t>(hidden.device().index()));
            if (refused.calls != 0 && kept + bytes >= refused.bytes) {
                --refused.calls;
            } else {
                try {
                    return LinearCrossEntropyStep::apply(flat, weight, indices, ignore_index, kind, static_cast<std::int64_t>(kept), static_cast<std::int64_t>(bytes));
                } catch (const c10::OutOfMemoryError&) { refused = RefusedWorkspace{kept + bytes, kAskAgainAfter}; }
            }
        }
    }
    const at::Tensor loss = LinearCrossEntropy::apply(flat, weight, indices, ignore_index, kind);
    return kind == FTCUDA_REDUCTION_NONE ? loss.view(target.sizes()) : loss;
}

}  // namespace

void registerLinearCrossEntropy(pybind11::module_& module) {
    module.def("linear_cross_entropy", &linearCrossEntropy,
               "Cross entropy of the logits hidden @ weight.T against `target`; an FP32 tensor.\n\n"
               "The logits are not kept. With a reduction and gradients wanted, their gradients wait for the backward pass where they take at most 2 GiB;\n"
               "otherwise, with recompute=True, or where there is no room for them, the backward pass computes the logits again, a piece of the vocabulary\n"
               "at a time, for a third more operations.\n"
               "hidden (..., depth) and weight (vocabulary, depth): FP32, FP16 or BF16, one type; target (...): INT64. Tokens whose target is\n"
               "ignore_index take no part, whatever their hidden state holds; any other target outside of the vocabulary gives NaN.\n"
               "reduction: 'mean' over the tokens that have a target (0 where none has), 'sum', or 'none' for a loss of target's shape.\n"
               "Differentiable once in hidden and weight; the gradients have their types.",
               pybind11::arg("hidden"), pybind11::arg("weight"), pybind11::arg("target"), pybind11::kw_only(), pybind11::arg("ignore_index") = -100,
               pybind11::arg("reduction") = "mean", pybind11::arg("recompute") = false);
}

}  // namespace flash_train_torch
