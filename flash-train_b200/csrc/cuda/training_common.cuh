// Shared by the operators of ftcuda/training.h: element types on the device, argument checks on the host.
#ifndef FTCUDA_TRAINING_COMMON_CUH_
#define FTCUDA_TRAINING_COMMON_CUH_

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "ftcuda/training.h"
#include "gemm_kernels.hpp"

namespace ftcuda {
namespace training {

template<typename T> struct Element;
template<> struct Element<float> {
    static constexpr int kCode = FTCUDA_ELEMENT_FP32;
    static __device__ __forceinline__ float widen(float x) { return x; }
    static __device__ __forceinline__ float narrow(float x) { return x; }
};
template<> struct Element<__half> {
    static constexpr int kCode = FTCUDA_ELEMENT_FP16;
    static __device__ __forceinline__ float widen(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half narrow(float x) { return __float2half_rn(x); }
};
template<> struct Element<__nv_bfloat16> {
    static constexpr int kCode = FTCUDA_ELEMENT_BF16;
    static __device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 narrow(float x) { return __float2bfloat16_rn(x); }
};

// An FP32 number as three BF16 ones, x = h + m + l to within its own rounding. A number that BF16 would round to infinity has the largest
// finite h; an infinity has that too, and itself in l, which meets the other operand's h alone in a product: the result is the
// infinity that FP32 arithmetic gives, or NaN against zero.
__device__ __forceinline__ void splitPlanes(float x, float (&parts)[3]) {
    constexpr float kLargest = 3.38953138925153547590e38F;
    float high = __bfloat162float(__float2bfloat16_rn(x));
    if (fabsf(high) > kLargest) { high = copysignf(kLargest, x); }
    const float rest   = x - high;
    const float middle = __bfloat162float(__float2bfloat16_rn(rest));
    const bool bounded = fabsf(rest) <= kLargest;
    parts[0]           = high;
    parts[1]           = bounded ? middle : 0.0F;
    parts[2]           = bounded ? rest - middle : rest;
}

// Bytes of an element, 0 for a type that the operators do not take.
inline std::uint64_t elementBytes(std::int32_t element) {
    return element == FTCUDA_ELEMENT_FP32 ? 4 : element == FTCUDA_ELEMENT_FP16 || element == FTCUDA_ELEMENT_BF16 ? 2 : 0;
}

inline bool aligned(const void* pointer, std::uint64_t bytes) { return reinterpret_cast<std::uintptr_t>(pointer) % bytes == 0; }

// Memory of one operand: `rows` windows of `width` bytes, `stride` bytes apart.
struct Range {
    std::uint64_t begin, end, width, stride;
};

inline Range rangeOf(const void* address, std::uint64_t rows, std::uint64_t cols, std::int64_t row_stride, std::uint64_t bytes) {
    Range r;
    r.begin  = reinterpret_cast<std::uintptr_t>(address);
    r.width  = cols * bytes;
    r.stride = rows > 1 ? static_cast<std::uint64_t>(row_stride) * bytes : 0;
    r.end    = r.begin + (rows - 1) * r.stride + r.width;
    return r;
}

// Whether two ranges whose hulls meet, the second beginning no earlier, share no byte as far as their strides show: windows of one matrix, side by side.
inline bool sideBySide(const Range& a, const Range& b) {
    const std::uint64_t stride = a.stride != 0 ? a.stride : b.stride;
    if (stride == 0 || (a.stride != 0 && b.stride != 0 && a.stride != b.stride) || a.width > stride || b.width > stride) { return false; }
    const std::uint64_t offset = (b.begin - a.begin) % stride;
    return offset >= a.width && offset + b.width <= stride;
}

// Whether they may share one, whichever begins earlier.
inline bool meet(const Range& a, const Range& b) {
    return a.begin < b.end && b.begin < a.end && !(a.begin <= b.begin ? sideBySide(a, b) : sideBySide(b, a));
}

// The device exists and is the calling thread's current one.
inline bool deviceIsCurrent(std::int32_t device, char* message, std::size_t capacity) {
    int current             = -1;
    const cudaError_t error = cudaGetDevice(&current);
    if (error != cudaSuccess) {
        fail(message, capacity, 1, "%s", cudaGetErrorString(error));
        return false;
    }
    if (current != device) {
        fail(message, capacity, 1, "device %d must be current, device %d is", device, current);
        return false;
    }
    return true;
}

// A kernel launch; `overlapped`: one that may start while the stream's preceding kernel ends (which the kernel waits for by gridDependencyWait).
template<typename... Parameters, typename... Arguments>
cudaError_t launchKernel(bool overlapped, void (*kernel)(Parameters...), dim3 grid, dim3 block, std::size_t shared, cudaStream_t stream,
                         const Arguments&... arguments) {
    cudaLaunchConfig_t config{};
    config.gridDim          = grid;
    config.blockDim         = block;
    config.dynamicSmemBytes = shared;
    config.stream           = stream;
    cudaLaunchAttribute attribute{};
    attribute.id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs                                         = &attribute;
    config.numAttrs                                      = overlapped ? 1 : 0;
    const cudaError_t error = cudaLaunchKernelEx(&config, kernel, arguments...);
    if (error == cudaSuccess) { countLaunches(1); }
    return error;
}

template<typename... Parameters, typename... Arguments>
cudaError_t launchOverlapped(void (*kernel)(Parameters...), dim3 grid, dim3 block, std::size_t shared, cudaStream_t stream,
                             const Arguments&... arguments) {
    return launchKernel(true, kernel, grid, block, shared, stream, arguments...);
}

}  // namespace training
}  // namespace ftcuda

#endif
