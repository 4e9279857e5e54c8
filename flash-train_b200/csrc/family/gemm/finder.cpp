#include "family/gemm/finder.hpp"

#include "cuda/gemm_choice.hpp"
#include "ftcuda/ftcuda.h"
#include "primitive/cuda/gemm/cuda_gemm.hpp"

namespace ftrain {

bool preparedFormPays(const GemmShape& shape) noexcept { return ftcuda::preparedFormPays(shape.m, shape.n, shape.k); }

std::vector<std::string> B200Heuristic::findCandidates(const GemmProblem& problem, const Constraints& constraints) {
    const GemmShape shape = problem.getShape();
    std::int32_t sms      = 148;
    if (ftcuda_device_sm_count(constraints.getDeviceId(), &sms, nullptr, 0) != 0 || sms <= 0) { sms = 148; }
    const bool b_along_k              = problem.getLayout(GemmPort::kB).row_stride == 1 && shape.n > 1;
    const ftcuda::GemmCandidates best = ftcuda::gemmCandidates(shape.m, shape.n, shape.k, b_along_k, static_cast<std::uint64_t>(sms));
    std::vector<std::string> names;
    for (int i = 0; i < best.count; ++i) { names.emplace_back(cudaGemmName(best.kernels[i])); }
    return names;
}

}  // namespace ftrain
