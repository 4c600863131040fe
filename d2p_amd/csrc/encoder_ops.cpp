// encoder_ops.cpp -- PyTorch registration of the sequence-encoder operators (namespace
// d2p_amd; no counterpart in the reference).
//
// As in torch_ops.cpp, every implementation validates on the host, allocates outputs and
// workspaces through the torch caching allocator and calls the C ABI on the current HIP
// stream.  d2p_amd::attention and d2p_amd::qk_norm_rope differentiate; the operators that
// do the work (attention_forward, attention_backward, qk_norm_rope_backward) go through
// the dispatcher, so that fake tensors reach their fakes when a compiler traces.
#include "encoder_util.h"

#include <ATen/autocast_mode.h>

#include <cmath>
#include <tuple>

namespace {

void check_4d(const Tensor& t, const Tensor& like, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.dim() == 4, name, " must be 4D (batch, length, heads, features), got ",
                t.dim(), "D");
    TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " must have q's type ",
                like.scalar_type(), ", got ", t.scalar_type());
    TORCH_CHECK(t.device() == like.device(), name, " must be on same device as q, got ",
                t.device(), " vs ", like.device());
}

void check_small(const Tensor& t, const Tensor& like, at::ScalarType type, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
    TORCH_CHECK(t.device() == like.device(), name, " must be on same device as q, got ",
                t.device(), " vs ", like.device());
}

d2p_strides strides_of(const Tensor& t) {
    // where there is one of something, its stride says nothing
    return {t.size(0) > 1 ? t.stride(0) : 0, t.size(1) > 1 ? t.stride(1) : t.size(3),
            t.size(2) > 1 ? t.stride(2) : 0};
}

// A tensor that the attention kernels can read: features adjacent, 16-byte rows that do not
// overlap.  Anything else is copied.
Tensor readable(const Tensor& t) {
    if (t.numel() == 0) return t;
    const int64_t per = 16 / t.element_size();
    const d2p_strides s = strides_of(t);
    const bool ok = (t.size(3) == 1 || t.stride(3) == 1) && s.batch % per == 0 &&
                    s.row % per == 0 && s.head % per == 0 && s.row >= t.size(3) &&
                    s.row * t.element_size() < (int64_t(1) << 31) / 128 &&
                    (uintptr_t)t.data_ptr() % 16 == 0;
    if (ok) return t;
    Tensor c = t.contiguous();
    return (uintptr_t)c.data_ptr() % 16 == 0 ? c : c.clone();
}

Tensor adjacent(const Tensor& t) {
    return t.size(3) == 1 || t.stride(3) == 1 ? t : t.contiguous();
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
d2p_attention_params attention_params(const Tensor& q, const Tensor& k, const Tensor& v,
                                      const OptTensor& lengths, bool causal, double scale,
                                      const OptTensor& bias, const OptTensor& buckets,
                                      double dropout, int64_t seed, const OptTensor& seed_tensor) {
    d2p_attention_params p{};
    TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
    p.dtype = type_code(q, "q");
    check_4d(q, q, "q");
    check_4d(k, q, "k");
    check_4d(v, q, "v");
    TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have the same shape, got ", k.sizes(),
                " and ", v.sizes());
    TORCH_CHECK(q.size(0) == k.size(0), "q and k must have the same batch size, got ", q.size(0),
                " and ", k.size(0));
    TORCH_CHECK(q.size(3) == k.size(3), "q and k must have the same head size, got ", q.size(3),
                " and ", k.size(3));
    TORCH_CHECK(q.size(3) >= 8 && q.size(3) <= 128 && q.size(3) % 8 == 0,
                "head size must be a multiple of 8 from 8 to 128, got ", q.size(3));
    TORCH_CHECK(k.size(2) >= 1 && q.size(2) >= 1 && q.size(2) % k.size(2) == 0,
                "query heads must be a positive multiple of key heads, got ", q.size(2), " and ",
                k.size(2));
    p.B = dim32(q.size(0), "batch size");
    p.Lq = dim32(q.size(1), "query length");
    p.Lk = dim32(k.size(1), "key length");
    p.Hq = dim32(q.size(2), "query heads");
    p.Hkv = dim32(k.size(2), "key heads");
    p.D = (int)q.size(3);
    p.q = strides_of(q);
    p.k = strides_of(k);
    p.v = strides_of(v);
    if (given(lengths)) {
        check_small(*lengths, q, torch::kInt32, "lengths");
        TORCH_CHECK(lengths->dim() == 2 && lengths->size(0) == p.B && lengths->size(1) == 2,
                    "lengths must be [B, 2] with B = ", p.B, ", got ", lengths->sizes());
        p.lengths = lengths->data_ptr<int>();
    }
    p.causal = causal;
    TORCH_CHECK(scale > 0 && std::isfinite(scale), "scale must be positive, got ", scale);
    p.scale = (float)scale;
    TORCH_CHECK(given(bias) == given(buckets), "bias and buckets go together");
    if (given(bias)) {
        TORCH_CHECK(bias->dim() == 2 && bias->size(0) >= 1 && bias->size(1) == p.Hq,
                    "bias must be [num_buckets, query heads] with ", p.Hq, " heads, got ",
                    bias->sizes());
        TORCH_CHECK(bias->scalar_type() == torch::kFloat32 ||
                        bias->scalar_type() == q.scalar_type(),
                    "bias must be float32 or of q's type, got ", bias->scalar_type());
        check_small(*bias, q, bias->scalar_type(), "bias");
        check_small(*buckets, q, torch::kInt32, "buckets");
        TORCH_CHECK(buckets->dim() == 1 && buckets->size(0) % 2 == 1 && buckets->size(0) <= 2049,
                    "buckets must be [2 R + 1], R at most 1024, got ", buckets->sizes());
        p.bias = bias->data_ptr();
        p.bias_dtype = type_code(*bias, "bias");
        p.num_buckets = dim32(bias->size(0), "buckets");
        p.buckets = buckets->data_ptr<int>();
        p.max_distance = (int)(buckets->size(0) / 2);
    }
    TORCH_CHECK(dropout >= 0 && dropout < 1, "dropout must be in [0, 1), got ", dropout);
    p.drop = (int)std::nearbyint(dropout * 256);
    TORCH_CHECK(dropout == 0 || (p.drop >= 1 && p.drop <= 255),
                "dropout is held in 256ths: between 1/512 and 511/512, got ", dropout);
    p.seed = (unsigned long long)seed;
    if (given(seed_tensor)) {
        check_small(*seed_tensor, q, torch::kInt64, "seed");
        TORCH_CHECK(seed_tensor->numel() == 1, "seed must hold one number");
        p.seed_ptr = (const long long*)seed_tensor->data_ptr<int64_t>();
    }
    return p;
}

std::tuple<Tensor, Tensor> attention_forward(const Tensor& q_, const Tensor& k_, const Tensor& v_,
                                             const OptTensor& lengths, bool causal, double scale,
                                             const OptTensor& bias, const OptTensor& buckets,
                                             double dropout, int64_t seed,
                                             const OptTensor& seed_tensor) {
    TORCH_CHECK(q_.is_cuda(), "q must be a CUDA tensor");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(q_.device());
    // sizes and types are checked before anything is copied
    auto p = attention_params(q_, k_, v_, lengths, causal, scale, bias, buckets, dropout, seed,
                              seed_tensor);
    const Tensor q = readable(q_), k = readable(k_), v = readable(v_);
    p.q = strides_of(q);
    p.k = strides_of(k);
    p.v = strides_of(v);
    Tensor out = torch::empty(q.sizes(), q.options());
    Tensor stats = torch::empty({2, p.B, p.Hq, p.Lq}, q.options().dtype(torch::kFloat32));
    const size_t bytes = d2p_attention_workspace_bytes(&p);
    Tensor ws;
    if (bytes) ws = workspace(bytes, q);
    D2P_CALL(d2p_attention_forward(&p, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                   stats.data_ptr<float>(), bytes ? ws.data_ptr() : nullptr, bytes,
                                   current_stream()));
    return {out, stats};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> attention_backward(
    const Tensor& grad_, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& out_,
    const Tensor& stats, const OptTensor& lengths, bool causal, double scale,
    const OptTensor& bias, const OptTensor& buckets, double dropout, int64_t seed,
    const OptTensor& seed_tensor, bool bias_grad) {
    TORCH_CHECK(q_.is_cuda(), "q must be a CUDA tensor");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(q_.device());
    auto p = attention_params(q_, k_, v_, lengths, causal, scale, bias, buckets, dropout, seed,
                              seed_tensor);
    check_4d(grad_, q_, "grad");
    check_4d(out_, q_, "out");
    TORCH_CHECK(grad_.sizes() == q_.sizes() && out_.sizes() == q_.sizes(),
                "grad and out must have q's shape, got ", grad_.sizes(), " and ", out_.sizes());
    check_small(stats, q_, torch::kFloat32, "stats");
    TORCH_CHECK(stats.numel() == 2 * q_.size(0) * q_.size(1) * q_.size(2),
                "stats must be [2, B, heads, queries], got ", stats.sizes());
    TORCH_CHECK(!bias_grad || given(bias), "a bias gradient needs a bias");
    const Tensor q = readable(q_), k = readable(k_), v = readable(v_), grad = readable(grad_);
    const Tensor out = out_.contiguous();
    p.q = strides_of(q);
    p.k = strides_of(k);
    p.v = strides_of(v);
    p.grad = strides_of(grad);
    Tensor dq = torch::empty(q.sizes(), q.options()), dk = torch::empty(k.sizes(), k.options()),
           dv = torch::empty(v.sizes(), v.options());
    Tensor db = bias_grad ? torch::empty(bias->sizes(), bias->options())
                          : torch::empty({0}, q.options());
    const size_t bytes = d2p_attention_backward_workspace_bytes(&p);
    Tensor ws = workspace(bytes, q);
    D2P_CALL(d2p_attention_backward(&p, grad.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                    out.data_ptr(), stats.data_ptr<float>(), dq.data_ptr(),
                                    dk.data_ptr(), dv.data_ptr(),
                                    bias_grad ? db.data_ptr() : nullptr, ws.data_ptr(), bytes,
                                    current_stream()));
    return {dq, dk, dv, db};
}

auto call_forward(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lengths,
                  bool causal, double scale, const OptTensor& bias, const OptTensor& buckets,
                  double dropout, int64_t seed, const OptTensor& seed_tensor) {
    static auto op = operator_handle<decltype(attention_forward)>("d2p_amd::attention_forward");
    return op.call(q, k, v, lengths, causal, scale, bias, buckets, dropout, seed, seed_tensor);
}

class AttentionFunction : public torch::autograd::Function<AttentionFunction> {
   public:
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                          const OptTensor& lengths, bool causal, double scale,
                          const OptTensor& bias, const OptTensor& buckets, double dropout,
                          int64_t seed, const OptTensor& seed_tensor) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [out, stats] = call_forward(q, k, v, lengths, causal, scale, bias, buckets, dropout,
                                         seed, seed_tensor);
        ctx->save_for_backward({q, k, v, out, stats, lengths.value_or(Tensor()),
                                bias.value_or(Tensor()), buckets.value_or(Tensor()),
                                seed_tensor.value_or(Tensor())});
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["dropout"] = dropout;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["bias"] = given(bias) && bias->requires_grad();
        return out;
    }
    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const auto s = ctx->get_saved_variables();
        const bool bias_grad = ctx->saved_data["bias"].toBool();
        no_tangents("attention's backward", {&grads[0]});
        BelowAutograd below;
        static auto op = operator_handle<decltype(attention_backward)>("d2p_amd::attention_backward");
        auto [dq, dk, dv, db] = op.call(
            grads[0], s[0], s[1], s[2], s[3], s[4], saved(s[5]), ctx->saved_data["causal"].toBool(),
            ctx->saved_data["scale"].toDouble(), saved(s[6]), saved(s[7]),
            ctx->saved_data["dropout"].toDouble(), ctx->saved_data["seed"].toInt(), saved(s[8]),
            bias_grad);
        return {dq, dk, dv, Tensor(), Tensor(), Tensor(), bias_grad ? db : Tensor(),
                Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lengths,
                 bool causal, double scale, const OptTensor& bias, const OptTensor& buckets,
                 double dropout, int64_t seed, const OptTensor& seed_tensor) {
    return std::get<0>(attention_forward(q, k, v, lengths, causal, scale, bias, buckets, dropout,
                                         seed, seed_tensor));
}

Tensor attention_autograd(const Tensor& q, const Tensor& k, const Tensor& v,
                          const OptTensor& lengths, bool causal, double scale,
                          const OptTensor& bias, const OptTensor& buckets, double dropout,
                          int64_t seed, const OptTensor& seed_tensor) {
    const Tensor b = bias.value_or(Tensor());
    no_tangents("attention", {&q, &k, &v, &b});
    if (differentiates({&q, &k, &v, &b}))
        return AttentionFunction::apply(q, k, v, lengths, causal, scale, bias, buckets, dropout,
                                        seed, seed_tensor);
    at::AutoDispatchBelowADInplaceOrView below;
    return std::get<0>(call_forward(q, k, v, lengths, causal, scale, bias, buckets, dropout, seed,
                                    seed_tensor));
}

// Under torch.autocast the products run in its type.
Tensor attention_autocast(const Tensor& q, const Tensor& k, const Tensor& v,
                          const OptTensor& lengths, bool causal, double scale,
                          const OptTensor& bias, const OptTensor& buckets, double dropout,
                          int64_t seed, const OptTensor& seed_tensor) {
    c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::Autocast);
    const auto type = at::autocast::get_autocast_dtype(at::kCUDA);
    static auto op = operator_handle<decltype(attention)>("d2p_amd::attention");
    OptTensor b = bias;
    if (given(bias) && bias->scalar_type() != torch::kFloat32)
        b = at::autocast::cached_cast(type, *bias);
    return op.call(at::autocast::cached_cast(type, q), at::autocast::cached_cast(type, k),
                   at::autocast::cached_cast(type, v), lengths, causal, scale, b, buckets, dropout,
                   seed, seed_tensor);
}

// ---------------------------------------------------------------------------
// norm and rotation of queries and keys
// ---------------------------------------------------------------------------
struct NormInputs {
    d2p_qk_norm_rope_params p{};
    Tensor q, k, wq, wk, cos, sin, positions;   // as the kernels read them
};

Tensor weight(const OptTensor& w, const Tensor& q, const char* name) {
    if (!given(w)) return Tensor();
    TORCH_CHECK(w->is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(w->device() == q.device(), name, " must be on same device as q, got ",
                w->device(), " vs ", q.device());
    TORCH_CHECK(w->dim() == 1 && w->size(0) == q.size(3), name, " must be [", q.size(3),
                "], got ", w->sizes());
    type_code(*w, name);
    return w->to(torch::kFloat32).contiguous();
}

NormInputs norm_inputs(const Tensor& q, const Tensor& k, const OptTensor& q_weight,
                       const OptTensor& k_weight, const Tensor& cos, const Tensor& sin,
                       const OptTensor& positions, double eps, bool interleaved) {
    NormInputs in;
    auto& p = in.p;
    TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
    p.dtype = type_code(q, "q");
    check_4d(q, q, "q");
    check_4d(k, q, "k");
    TORCH_CHECK(q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3),
                "q and k must have the same batch size, length and head size, got ", q.sizes(),
                " and ", k.sizes());
    TORCH_CHECK(q.size(3) >= 8 && q.size(3) <= 128 && q.size(3) % 8 == 0,
                "head size must be a multiple of 8 from 8 to 128, got ", q.size(3));
    TORCH_CHECK(cos.dim() == 2 && cos.sizes() == sin.sizes(),
                "cos and sin must be [positions, rotated features / 2] both, got ", cos.sizes(),
                " and ", sin.sizes());
    check_small(cos, q, torch::kFloat32, "cos");
    check_small(sin, q, torch::kFloat32, "sin");
    TORCH_CHECK(2 * cos.size(1) <= q.size(3), "cos and sin rotate at most the head size, got ",
                2 * cos.size(1), " of ", q.size(3));
    TORCH_CHECK(eps >= 0, "eps must not be negative, got ", eps);
    p.B = dim32(q.size(0), "batch size");
    p.L = dim32(q.size(1), "length");
    p.Hq = dim32(q.size(2), "query heads");
    p.Hkv = dim32(k.size(2), "key heads");
    p.D = (int)q.size(3);
    p.R = (int)(2 * cos.size(1));
    in.q = adjacent(q);
    in.k = adjacent(k);
    p.q = strides_of(in.q);
    p.k = strides_of(in.k);
    in.wq = weight(q_weight, q, "q_weight");
    in.wk = weight(k_weight, q, "k_weight");
    in.cos = cos;
    in.sin = sin;
    p.q_weight = in.wq.defined() ? in.wq.data_ptr<float>() : nullptr;
    p.k_weight = in.wk.defined() ? in.wk.data_ptr<float>() : nullptr;
    p.cos = cos.data_ptr<float>();
    p.sin = sin.data_ptr<float>();
    p.table_rows = cos.size(0);
    if (given(positions)) {
        check_small(*positions, q, torch::kInt32, "positions");
        TORCH_CHECK(positions->dim() == 2 && positions->size(0) == p.B &&
                        positions->size(1) == p.L,
                    "positions must be [B, L] = [", p.B, ", ", p.L, "], got ", positions->sizes());
        p.positions = positions->data_ptr<int>();
        in.positions = *positions;
    } else {
        TORCH_CHECK(p.R == 0 || p.table_rows >= p.L, "cos and sin must have a row for each of ",
                    p.L, " positions, got ", p.table_rows);
    }
    p.eps = (float)eps;
    p.interleaved = interleaved;
    return in;
}

std::tuple<Tensor, Tensor> qk_norm_rope_run(const Tensor& q, const Tensor& k,
                                            const OptTensor& q_weight, const OptTensor& k_weight,
                                            const Tensor& cos, const Tensor& sin,
                                            const OptTensor& positions, double eps,
                                            bool interleaved) {
    TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
    const auto in = norm_inputs(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved);
    Tensor oq = torch::empty(q.sizes(), q.options()), ok = torch::empty(k.sizes(), k.options());
    D2P_CALL(d2p_qk_norm_rope(&in.p, in.q.data_ptr(), in.k.data_ptr(), oq.data_ptr(),
                              ok.data_ptr(), current_stream()));
    return {oq, ok};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> qk_norm_rope_backward(
    const Tensor& gq_, const Tensor& gk_, const Tensor& q, const Tensor& k,
    const OptTensor& q_weight, const OptTensor& k_weight, const Tensor& cos, const Tensor& sin,
    const OptTensor& positions, double eps, bool interleaved, bool weight_grads) {
    TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
    auto in = norm_inputs(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved);
    check_4d(gq_, q, "grad of q");
    check_4d(gk_, q, "grad of k");
    TORCH_CHECK(gq_.sizes() == q.sizes() && gk_.sizes() == k.sizes(),
                "gradients must have the shapes of q and k");
    const Tensor gq = adjacent(gq_), gk = adjacent(gk_);
    in.p.gq = strides_of(gq);
    in.p.gk = strides_of(gk);
    Tensor dq = torch::empty(q.sizes(), q.options()), dk = torch::empty(k.sizes(), k.options());
    const auto f32 = q.options().dtype(torch::kFloat32);
    Tensor dwq = torch::empty({weight_grads ? q.size(3) : 0}, f32), dwk = torch::empty_like(dwq);
    const size_t bytes = weight_grads ? d2p_qk_norm_rope_backward_workspace_bytes(&in.p) : 0;
    Tensor ws = workspace(bytes, q);
    D2P_CALL(d2p_qk_norm_rope_backward(&in.p, gq.data_ptr(), gk.data_ptr(), in.q.data_ptr(),
                                       in.k.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                                       weight_grads ? dwq.data_ptr<float>() : nullptr,
                                       weight_grads ? dwk.data_ptr<float>() : nullptr,
                                       ws.data_ptr(), bytes, current_stream()));
    return {dq, dk, dwq, dwk};
}

auto call_norm(const Tensor& q, const Tensor& k, const OptTensor& q_weight,
               const OptTensor& k_weight, const Tensor& cos, const Tensor& sin,
               const OptTensor& positions, double eps, bool interleaved) {
    static auto op = operator_handle<decltype(qk_norm_rope_run)>("d2p_amd::qk_norm_rope");
    return op.call(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved);
}

class QkNormRopeFunction : public torch::autograd::Function<QkNormRopeFunction> {
   public:
    static tensor_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k,
                               const OptTensor& q_weight, const OptTensor& k_weight,
                               const Tensor& cos, const Tensor& sin, const OptTensor& positions,
                               double eps, bool interleaved) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [oq, ok] = call_norm(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved);
        ctx->save_for_backward({q, k, q_weight.value_or(Tensor()), k_weight.value_or(Tensor()),
                                cos, sin, positions.value_or(Tensor())});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["weights"] = (given(q_weight) && q_weight->requires_grad()) ||
                                     (given(k_weight) && k_weight->requires_grad());
        return {oq, ok};
    }
    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const auto s = ctx->get_saved_variables();
        const bool weights = ctx->saved_data["weights"].toBool();
        no_tangents("qk_norm_rope's backward", {&grads[0], &grads[1]});
        BelowAutograd below;
        static auto op =
            operator_handle<decltype(qk_norm_rope_backward)>("d2p_amd::qk_norm_rope_backward");
        auto [dq, dk, dwq, dwk] = op.call(
            grads[0], grads[1], s[0], s[1], saved(s[2]), saved(s[3]), s[4], s[5], saved(s[6]),
            ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool(), weights);
        auto grad_of = [&](const Tensor& w, const Tensor& dw) {
            return weights && w.defined() ? dw.to(w.scalar_type()) : Tensor();
        };
        return {dq, dk, grad_of(s[2], dwq), grad_of(s[3], dwk), Tensor(), Tensor(), Tensor(),
                Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> qk_norm_rope_autograd(const Tensor& q, const Tensor& k,
                                                 const OptTensor& q_weight,
                                                 const OptTensor& k_weight, const Tensor& cos,
                                                 const Tensor& sin, const OptTensor& positions,
                                                 double eps, bool interleaved) {
    const Tensor wq = q_weight.value_or(Tensor()), wk = k_weight.value_or(Tensor());
    no_tangents("qk_norm_rope", {&q, &k, &wq, &wk, &cos, &sin});
    TORCH_CHECK(!differentiates({&cos, &sin}), "cos and sin do not take gradients");
    if (differentiates({&q, &k, &wq, &wk})) {
        auto r = QkNormRopeFunction::apply(q, k, q_weight, k_weight, cos, sin, positions, eps,
                                           interleaved);
        return {r[0], r[1]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return call_norm(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved);
}

}  // namespace

#define ATTENTION_OPTIONS                                                                   \
    "Tensor? lengths, bool causal, float scale, Tensor? bias, Tensor? buckets, "            \
    "float dropout, int seed, Tensor? seed_tensor"
#define NORM_OPTIONS                                                                        \
    "Tensor? q_weight, Tensor? k_weight, Tensor cos, Tensor sin, Tensor? positions, "       \
    "float eps, bool interleaved"

TORCH_LIBRARY_FRAGMENT(d2p_amd, m) {
    m.def("attention(Tensor q, Tensor k, Tensor v, " ATTENTION_OPTIONS ") -> Tensor");
    m.def("attention_forward(Tensor q, Tensor k, Tensor v, " ATTENTION_OPTIONS
          ") -> (Tensor, Tensor)");
    m.def("attention_backward(Tensor grad, Tensor q, Tensor k, Tensor v, Tensor out, "
          "Tensor stats, " ATTENTION_OPTIONS ", bool bias_grad) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("qk_norm_rope(Tensor q, Tensor k, " NORM_OPTIONS ") -> (Tensor, Tensor)");
    m.def("qk_norm_rope_backward(Tensor gq, Tensor gk, Tensor q, Tensor k, " NORM_OPTIONS
          ", bool weight_grads) -> (Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(d2p_amd, CUDA, m) {
    m.impl("attention", attention);
    m.impl("attention_forward", attention_forward);
    m.impl("attention_backward", attention_backward);
    m.impl("qk_norm_rope", qk_norm_rope_run);
    m.impl("qk_norm_rope_backward", qk_norm_rope_backward);
}

// The operators below the differentiable ones have no gradients of their own: a second
// derivative raises.
TORCH_LIBRARY_IMPL(d2p_amd, Autograd, m) {
    m.impl("attention", attention_autograd);
    m.impl("qk_norm_rope", qk_norm_rope_autograd);
    m.impl("attention_forward", torch::autograd::autogradNotImplementedFallback());
    m.impl("attention_backward", torch::autograd::autogradNotImplementedFallback());
    m.impl("qk_norm_rope_backward", torch::autograd::autogradNotImplementedFallback());
}

TORCH_LIBRARY_IMPL(d2p_amd, AutocastCUDA, m) { m.impl("attention", attention_autocast); }

TORCH_LIBRARY_IMPL(d2p_amd, CPU, m) {
    for (const char* name : {"attention", "attention_forward", "attention_backward",
                             "qk_norm_rope", "qk_norm_rope_backward"})
        m.impl(name, torch::CppFunction::makeFromBoxedFunction<&cpu_boxed>());
}
