// encoder_util.h -- what the operator layers of the sequence encoder share: types, sizes, the
// rules of their autograd functions.
#pragma once
#include "torch_util.h"

#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>

#include <limits>

#include "../../include/d2p_amd_encoder.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;
using OptTensor = c10::optional<Tensor>;

inline bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

inline int type_code(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case torch::kFloat32: return D2P_FLOAT32;
        case torch::kFloat16: return D2P_FLOAT16;
        case torch::kBFloat16: return D2P_BFLOAT16;
        default:
            TORCH_CHECK(false, name, " must be float32, float16 or bfloat16, got ",
                        t.scalar_type());
    }
}

inline int dim32(int64_t v, const char* what) {
    TORCH_CHECK(v <= std::numeric_limits<int>::max(), what, " must fit int32, got ", v);
    return (int)v;
}

template <class F> auto operator_handle(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

// A backward pass that nobody differentiates skips the autograd layer of the operators it
// calls; in one that somebody does, that layer makes their derivative raise.
struct BelowAutograd {
    c10::optional<at::AutoDispatchBelowADInplaceOrView> guard;
    BelowAutograd() {
        if (!at::GradMode::is_enabled()) guard.emplace();
    }
};

// Forward-mode derivatives are not implemented: a tangent raises, with and without gradients.
inline void no_tangents(const char* name, std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), name,
                                    " does not support forward AD");
}

inline OptTensor saved(const Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }

inline bool differentiates(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

}  // namespace
