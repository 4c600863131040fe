// attention.hip -- the C ABI of attention (include/d2p_amd_encoder.h).
#include <algorithm>

#include "attention_backward.hip.h"
#include "attention_few.hip.h"

namespace d2p_amd {
namespace enc {

static int check_strides(const d2p_strides& s, int rows, int D, int dtype, const char* name) {
    const int per = dtype == D2P_FLOAT32 ? 4 : 8;   // elements of 16 bytes
    if (s.batch % per || s.row % per || s.head % per) {
        set_last_error("%s: strides must be multiples of 16 bytes", name);
        return D2P_ERR_ARG;
    }
    if (s.batch < 0 || s.row < 0 || s.head < 0 || (rows > 1 && s.row < D)) {
        set_last_error("%s: strides must not be negative, and rows must not overlap", name);
        return D2P_ERR_ARG;
    }
    if (s.row * type_bytes(dtype) >= (1LL << 31) / 128) {
        set_last_error("%s: 128 rows must span less than 2 GiB", name);
        return D2P_ERR_ARG;
    }
    return D2P_OK;
}

// Every argument of an attention call that the host can see.
static int check_attention(const d2p_attention_params* p) {
    D2P_REQUIRE(p != nullptr, "null parameters");
    D2P_REQUIRE(p->dtype == D2P_FLOAT32 || p->dtype == D2P_FLOAT16 || p->dtype == D2P_BFLOAT16,
                "unknown element type");
    D2P_REQUIRE(p->B >= 0 && p->Lq >= 0 && p->Lk >= 0, "negative size");
    D2P_REQUIRE(p->Hq >= 1 && p->Hkv >= 1 && p->Hq % p->Hkv == 0,
                "query heads must be a positive multiple of key heads");
    D2P_REQUIRE(p->D >= 8 && p->D <= 128 && p->D % 8 == 0,
                "head size must be a multiple of 8 from 8 to 128");
    D2P_REQUIRE(p->Lq <= 0x7fffff00 && p->Lk <= 0x7fffff00 &&
                (long long)p->Lq + p->Lk <= 0x7fffff00, "sequences too long");
    D2P_REQUIRE((long long)p->B * p->Hq <= 0x7fffffff, "too many heads");
    D2P_REQUIRE(p->scale > 0.0f && p->scale < __builtin_inff(), "scale must be positive");
    D2P_REQUIRE(p->drop >= 0 && p->drop <= 255, "drop must be between 0 and 255");
    if (p->bias) {
        D2P_REQUIRE(p->bias_dtype == D2P_FLOAT32 || p->bias_dtype == p->dtype,
                    "bias must be float32 or of the inputs' type");
        D2P_REQUIRE(p->buckets && p->num_buckets >= 1, "bias needs buckets");
        D2P_REQUIRE(p->max_distance >= 0 && p->max_distance <= 1024,
                    "max_distance must be between 0 and 1024");
    }
    D2P_TRY(check_strides(p->q, p->Lq, p->D, p->dtype, "q"));
    D2P_TRY(check_strides(p->k, p->Lk, p->D, p->dtype, "k"));
    D2P_TRY(check_strides(p->v, p->Lk, p->D, p->dtype, "v"));
    return D2P_OK;
}

static bool aligned(const void* x) { return ((uintptr_t)x & 15) == 0; }

// Parts of the backward pass's workspace, in floats.
struct BackwardLayout {
    size_t heads, delta, partial, largest;
    explicit BackwardLayout(const d2p_attention_params& p) {
        // first, for its 16-byte accesses (D is a multiple of 8)
        heads = split_groups(p) ? 2 * (size_t)p.B * p.Lk * p.Hq * p.D : 0;
        delta = (size_t)p.B * p.Hq * p.Lq;
        partial = p.bias ? (size_t)p.B * p.Hq * query_blocks(p) * (2 * p.max_distance + 1) : 0;
        largest = p.dtype == D2P_FLOAT16 ? (size_t)p.B * p.Hq * query_blocks(p) * 4 : 0;
    }
    size_t bytes() const { return (heads + delta + partial + largest) * 4; }
};

}  // namespace enc
}  // namespace d2p_amd

using namespace d2p_amd;
using namespace d2p_amd::enc;

extern "C" size_t d2p_attention_workspace_bytes(const d2p_attention_params* p) {
    FewPlan pl;
    return p && check_attention(p) == D2P_OK && plan_few(*p, &pl) ? few_floats(*p, pl) * 4 : 0;
}

extern "C" int d2p_attention_forward(const d2p_attention_params* p, const void* q, const void* k,
                                     const void* v, void* out, float* stats, void* workspace,
                                     size_t workspace_bytes, void* stream) {
    D2P_TRY(check_attention(p));
    if (p->B == 0 || p->Lq == 0) return D2P_OK;
    D2P_REQUIRE(q && out && stats && ((k && v) || p->Lk == 0), "null pointer argument");
    D2P_REQUIRE(aligned(q) && aligned(k) && aligned(v) && aligned(out),
                "tensors must be aligned to 16 bytes");
    const ForwardArgs a{*p, q, k, v, out, stats};
    hipStream_t st = (hipStream_t)stream;
    FewArgs few{a};
    if (plan_few(*p, &few.plan)) {
        const size_t floats = few_floats(*p, few.plan);
        D2P_REQUIRE(floats == 0 || (workspace && workspace_bytes >= floats * 4),
                    "workspace too small");
        const size_t rows = (size_t)p->B * p->Hkv * few.plan.rows * few.plan.parts;
        few.acc = (float*)workspace;
        few.part_m = few.acc + rows * p->D;
        few.part_l = few.part_m + rows;
        return p->dtype == D2P_FLOAT32   ? launch_few_f32(few, st)
               : p->dtype == D2P_FLOAT16 ? launch_few_f16(few, st)
                                         : launch_few_bf16(few, st);
    }
    return p->dtype == D2P_FLOAT32   ? launch_forward_f32(a, st)
           : p->dtype == D2P_FLOAT16 ? launch_forward_f16(a, st)
                                     : launch_forward_bf16(a, st);
}

extern "C" size_t d2p_attention_backward_workspace_bytes(const d2p_attention_params* p) {
    return p && p->B > 0 ? BackwardLayout(*p).bytes() : 0;
}

extern "C" int d2p_attention_backward(const d2p_attention_params* p, const void* grad,
                                      const void* q, const void* k, const void* v,
                                      const void* out, const float* stats, void* dq, void* dk,
                                      void* dv, void* dbias, void* workspace,
                                      size_t workspace_bytes, void* stream) {
    D2P_TRY(check_attention(p));
    D2P_TRY(check_strides(p->grad, p->Lq, p->D, p->dtype, "grad"));
    D2P_REQUIRE(!dbias || p->bias, "a bias gradient needs a bias");
    hipStream_t st = (hipStream_t)stream;
    if (p->B > 0) {
        D2P_REQUIRE((grad && q && out && stats && dq) || p->Lq == 0, "null pointer argument");
        D2P_REQUIRE((k && v && dk && dv) || p->Lk == 0, "null pointer argument");
        D2P_REQUIRE(aligned(grad) && aligned(q) && aligned(k) && aligned(v) && aligned(out) &&
                    aligned(dq) && aligned(dk) && aligned(dv),
                    "tensors must be aligned to 16 bytes");
    }
    const BackwardLayout lay(*p);
    D2P_REQUIRE(((uintptr_t)workspace & 15) == 0, "workspace must be aligned to 16 bytes");
    D2P_REQUIRE(lay.bytes() == 0 || (workspace && workspace_bytes >= lay.bytes()),
                "workspace too small");
    BackwardArgs a{*p, grad, q, k, v, out, stats, dq, dk, dv, dbias};
    a.heads = lay.heads ? (float*)workspace : nullptr;
    a.delta = (float*)workspace + lay.heads;
    a.partial = a.delta + lay.delta;
    a.largest = a.partial + lay.partial;
    if (p->B == 0 && !dbias) return D2P_OK;
    return p->dtype == D2P_FLOAT32   ? launch_backward_f32(a, st)
           : p->dtype == D2P_FLOAT16 ? launch_backward_f16(a, st)
                                     : launch_backward_bf16(a, st);
}
