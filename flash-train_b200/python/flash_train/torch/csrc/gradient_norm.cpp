// flash_train.torch.grad_norm and clip_grads over ftcuda_gradient_norm / ftcuda_gradient_clip.
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include <ftcuda/training.h>

#include "training.hpp"

namespace flash_train_torch {

at::Tensor workspaceFor(std::uint64_t bytes, const at::Tensor& like) {
    return at::empty({static_cast<std::int64_t>(bytes)}, like.options().dtype(at::kByte).requires_grad(false));
}

std::int32_t elementOf(const at::Tensor& tensor) {
    switch (tensor.scalar_type()) {
        case at::kFloat: return FTCUDA_ELEMENT_FP32;
        case at::kHalf: return FTCUDA_ELEMENT_FP16;
        case at::kBFloat16: return FTCUDA_ELEMENT_BF16;
        default: return 0;
    }
}

namespace {

void checkGradient(const at::Tensor& tensor, const at::Tensor& first, const char* name, std::size_t index) {
    TORCH_CHECK(tensor.is_cuda() && tensor.layout() == at::kStrided, name, " ", index, " must be a dense device tensor");
    TORCH_CHECK(elementOf(tensor) != 0, name, " ", index, " must be FP32, FP16 or BF16");
    TORCH_CHECK(tensor.device() == first.device(), name, " ", index, " must be on the first gradient's device");
    TORCH_CHECK(!tensor.is_neg(), name, " ", index, " must not be a negated view");
}

// Rows of neighbouring elements, whatever the order of the dimensions: those that both sides walk without a gap become one.
FtcudaGradient describe(const at::Tensor& gradient, const at::Tensor& out, std::size_t index) {
    FtcudaGradient g{};
    g.data        = gradient.data_ptr();
    g.out         = out.data_ptr();
    g.element     = elementOf(gradient);
    g.out_element = elementOf(out);
    if (gradient.numel() == 0) { return g; }
    if (gradient.is_contiguous() && out.is_contiguous()) {
        g.rows = 1;
        g.cols = static_cast<std::uint64_t>(gradient.numel());
        return g;
    }
    struct Dimension {
        std::int64_t size, stride, out_stride;
    };
    std::vector<Dimension> dimensions;
    for (std::int64_t d = 0; d < gradient.dim(); ++d) {
        if (gradient.size(d) != 1) { dimensions.push_back({gradient.size(d), gradient.stride(d), out.stride(d)}); }
    }
    std::stable_sort(dimensions.begin(), dimensions.end(), [](const Dimension& a, const Dimension& b) { return a.stride < b.stride; });
    std::vector<Dimension> merged{{1, 1, 1}};
    for (const Dimension& d : dimensions) {
        Dimension& last = merged.back();
        if (d.stride == last.size * last.stride && d.out_stride == last.size * last.out_stride) {
            last.size *= d.size;
        } else {
            merged.push_back(d);
        }
    }
    const bool sound = merged.size() == 1 || (merged.size() == 2 && merged[1].stride >= merged[0].size && merged[1].out_stride >= merged[0].size);
    TORCH_CHECK(sound, "gradient ", index, " (with its output) must be dense, or rows of neighbouring elements at equal distances");
    g.cols = static_cast<std::uint64_t>(merged[0].size);
    g.rows = 1;
    if (merged.size() == 2) {
        g.rows           = static_cast<std::uint64_t>(merged[1].size);
        g.row_stride     = merged[1].stride;
        g.out_row_stride = merged[1].out_stride;
    }
    return g;
}

int normKind(double norm_type) {
    TORCH_CHECK(norm_type == 2.0 || (std::isinf(norm_type) && norm_type > 0.0), "norm_type must be 2 or infinity");
    return norm_type == 2.0 ? FTCUDA_NORM_2 : FTCUDA_NORM_INF;
}

// The tensors of a Python sequence, looked at in place: with many small ones, what the host does for each is most of a call.
class TensorList final {
  public:
    TensorList(pybind11::handle sequence, const char* name) : items_(pybind11::reinterpret_steal<pybind11::object>(PySequence_Fast(sequence.ptr(), name))) {
        if (!items_) { throw pybind11::error_already_set(); }
        for (std::size_t i = 0; i < size(); ++i) { TORCH_CHECK(THPVariable_Check(item(i)), name, " ", i, " must be a tensor"); }
    }
    std::size_t size() const { return static_cast<std::size_t>(PySequence_Fast_GET_SIZE(items_.ptr())); }
    const at::Tensor& operator[](std::size_t i) const { return THPVariable_Unpack(item(i)); }

  private:
    PyObject* item(std::size_t i) const { return PySequence_Fast_GET_ITEM(items_.ptr(), static_cast<Py_ssize_t>(i)); }
    pybind11::object items_;  // a list or a tuple
};

at::Tensor normOf(const TensorList& gradients, const TensorList* outs, double norm_type, double max_norm) {
    const int kind = normKind(norm_type);
    TORCH_CHECK(outs == nullptr || max_norm >= 0.0, "max_norm must not be negative");
    if (gradients.size() == 0) { return at::zeros({}, at::kFloat); }
    const at::Tensor& first = gradients[0];
    std::vector<FtcudaGradient> described;
    described.reserve(gradients.size());
    const bool recording = at::GradMode::is_enabled();
    for (std::size_t i = 0; i < gradients.size(); ++i) {
        const at::Tensor& gradient = gradients[i];
        const at::Tensor& out      = outs != nullptr ? (*outs)[i] : gradient;
        checkGradient(gradient, first, "gradient", i);
        TORCH_CHECK(!recording || !gradient.requires_grad(), "gradient ", i, " must not require a gradient: the norm is not differentiable (detach it, or use torch.no_grad())");
        if (outs != nullptr) {
            if (!out.is_same(gradient)) {
                checkGradient(out, first, "out", i);
                TORCH_CHECK(out.sizes() == gradient.sizes(), "out ", i, " must have its gradient's shape");
            }
            TORCH_CHECK(!recording || !out.requires_grad(), "out ", i, " must not require a gradient");
        }
        described.push_back(describe(gradient, out, i));
    }
    const c10::cuda::CUDAGuard guard(first.device());
    const auto stream             = c10::cuda::getCurrentCUDAStream(first.device().index()).stream();
    at::Tensor norm               = at::empty({}, first.options().dtype(at::kFloat).requires_grad(false));
    const std::uint64_t bytes     = ftcuda_gradient_norm_workspace_bytes(described.size());
    const at::Tensor workspace    = workspaceFor(bytes, first);
    const std::int32_t device     = first.device().index();
    Message message;
    const int status = outs == nullptr ? ftcuda_gradient_norm(described.data(), described.size(), kind, norm.data_ptr<float>(), device, workspace.data_ptr(),
                                                              bytes, stream, message.text, sizeof message.text)
                                       : ftcuda_gradient_clip(described.data(), described.size(), kind, max_norm, norm.data_ptr<float>(), device,
                                                              workspace.data_ptr(), bytes, stream, message.text, sizeof message.text);
    TORCH_CHECK(status == 0, "flash_train ", outs == nullptr ? "grad_norm" : "clip_grads", " failed: ", message.text);
    for (std::size_t i = 0; outs != nullptr && i < outs->size(); ++i) {
        if (!(*outs)[i].is_inference()) { torch::autograd::impl::bump_version((*outs)[i]); }
    }
    return norm;
}

at::Tensor gradNorm(const pybind11::object& gradients, double norm_type) { return normOf(TensorList(gradients, "gradients"), nullptr, norm_type, 0.0); }

at::Tensor clipGrads(const pybind11::object& gradients, double max_norm, double norm_type, const pybind11::object& out) {
    const TensorList from(gradients, "gradients");
    if (out.is_none()) { return normOf(from, &from, norm_type, max_norm); }
    const TensorList to(out, "out");
    TORCH_CHECK(to.size() == from.size(), "out must have one tensor for each gradient");
    return normOf(from, &to, norm_type, max_norm);
}

}  // namespace

void registerGradientNorm(pybind11::module_& module) {
    module.def("grad_norm", &gradNorm,
               "Norm over all elements of a list of gradients (FP32, FP16, BF16; any sizes), as one FP32 number on their device.\n\n"
               "norm_type: 2, or infinity for the largest magnitude. Not differentiable: tensors that require a gradient are refused outside of torch.no_grad().",
               pybind11::arg("gradients"), pybind11::arg("norm_type") = 2.0);
    module.def("clip_grads", &clipGrads,
               "Multiplies every gradient by min(1, max_norm / (norm + 1e-6)) and returns the norm before that, without waiting for it.\n\n"
               "In place, or into `out`: tensors of the same shapes in any of the three types. Not differentiable, as grad_norm.",
               pybind11::arg("gradients"), pybind11::arg("max_norm"), pybind11::arg("norm_type") = 2.0, pybind11::arg("out") = pybind11::none());
}

}  // namespace flash_train_torch
