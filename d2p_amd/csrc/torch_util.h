// torch_util.h -- what the operator layer's files share: calls of the C ABI on the current
// HIP stream, workspaces from torch's caching allocator, the refusal of CPU tensors.
#pragma once
#include <torch/torch.h>
#include <torch/library.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <algorithm>

#include "../../include/d2p_amd.h"

#define D2P_CALL(expr)                                                          \
    do {                                                                        \
        int rc_ = (expr);                                                       \
        TORCH_CHECK(rc_ == 0, "d2p_amd kernel call failed: ", d2p_last_error()); \
    } while (0)

namespace {

inline void* current_stream() {
    return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream();
}

inline torch::Tensor workspace(size_t bytes, const torch::Tensor& like) {
    return torch::empty({(int64_t)std::max<size_t>(bytes, 1)},
                        like.options().dtype(torch::kUInt8));
}

[[noreturn]] inline void cpu_unsupported() {
    TORCH_CHECK(false,
                "d2p_amd implements the MI355X (HIP) path only: move the inputs to a "
                "HIP device (device='cuda' on PyTorch-ROCm)");
}

inline void cpu_boxed(const c10::OperatorHandle&, torch::jit::Stack*) { cpu_unsupported(); }

}  // namespace
