// The operators around a training step's products, registered beside gemm.
#ifndef FLASH_TRAIN_TORCH_TRAINING_HPP_
#define FLASH_TRAIN_TORCH_TRAINING_HPP_

#include <torch/extension.h>

#include <cstdint>
#include <vector>

namespace flash_train_torch {

void registerGradientNorm(pybind11::module_& module);
void registerExpertRouting(pybind11::module_& module);
void registerLinearCrossEntropy(pybind11::module_& module);

// Room for a reason from the library.
struct Message {
    char text[256] = "";
};

// A block of torch's caching allocator on `like`'s device. The allocator keeps it reserved for the current stream until the work enqueued so
// far is done, so it may go out of scope behind the call that got it.
at::Tensor workspaceFor(std::uint64_t bytes, const at::Tensor& like);

// A size that torch's allocator could not give a thread on a device, and for how many more calls nothing as large is asked
// for: each refusal makes the allocator synchronise the device and give back all that it caches, which a program near
// the end of the memory would pay on every call.
struct RefusedWorkspace {
    std::uint64_t bytes = 0;
    unsigned calls      = 0;
};
constexpr unsigned kAskAgainAfter = 64;

inline RefusedWorkspace& ofDevice(std::vector<RefusedWorkspace>& refused, std::size_t device) {
    if (refused.size() <= device) { refused.resize(device + 1); }
    return refused[device];
}

// FTCUDA_ELEMENT_* of a floating type that the operators take, 0 for any other.
std::int32_t elementOf(const at::Tensor& tensor);

}  // namespace flash_train_torch

#endif
