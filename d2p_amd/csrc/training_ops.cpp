// training_ops.cpp -- PyTorch registration of the operators around a sequence encoder's
// attention layers: token embedding, the residual stream's norms, gradient norm and clipping
// (namespace d2p_amd; no counterpart in the reference).
//
// Built as encoder_ops.cpp is: host checks, outputs and workspaces from torch's caching
// allocator, the C ABI on the current HIP stream; token_embedding and residual_norm
// differentiate, and the operators that do their work go through the dispatcher.
#include "encoder_util.h"

#include <ATen/MemoryOverlap.h>

#include <cmath>
#include <tuple>
#include <vector>

#include "../../include/d2p_amd_training.h"

namespace {

void check_on(const Tensor& t, const Tensor& like, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.device() == like.device(), name, " must be on same device as the others, got ",
                t.device(), " vs ", like.device());
}

// Strides of a [.., row, feature] tensor whose features are adjacent (a copy where they are not).
Tensor adjacent_rows(const Tensor& t) {
    return t.stride(-1) == 1 ? t : t.contiguous();
}
d2p_row_strides row_strides(const Tensor& t) {
    return {t.size(0) > 1 ? t.stride(0) : 0, t.size(1) > 1 ? t.stride(1) : 0};
}

// ---------------------------------------------------------------------------
// token embedding
// ---------------------------------------------------------------------------
struct EmbedInputs {
    d2p_token_embedding_params p{};
    Tensor tokens, lengths;
};

EmbedInputs embed_inputs(const Tensor& tokens, const OptTensor& lengths, double scale,
                         int64_t padding, int64_t rows, int64_t features, int weight_dtype,
                         int dtype) {
    EmbedInputs in;
    auto& p = in.p;
    TORCH_CHECK(tokens.is_cuda(), "tokens must be a CUDA tensor");
    TORCH_CHECK(tokens.scalar_type() == torch::kInt32 || tokens.scalar_type() == torch::kInt64,
                "tokens must be int32 or int64, got ", tokens.scalar_type());
    const bool batched = tokens.dim() == 2;
    p.B = batched ? dim32(tokens.size(0), "batch size") : 1;
    p.L = dim32(batched ? tokens.size(1) : tokens.numel(), "length");
    TORCH_CHECK((int64_t)p.B * p.L < int64_t(1) << 31, "too many tokens: ", tokens.numel());
    p.V = dim32(rows, "rows of the weight");
    p.D = dim32(features, "features");
    TORCH_CHECK(p.D >= 8 && p.D <= 1 << 20, "features must be between 8 and 2^20, got ", p.D);
    TORCH_CHECK(p.V >= 1 && p.V < std::numeric_limits<int>::max(),
                "weight must have between 1 and 2^31 - 2 rows, got ", p.V);
    p.weight_dtype = weight_dtype;
    p.dtype = dtype;
    TORCH_CHECK(weight_dtype == dtype || weight_dtype == D2P_FLOAT32,
                "embeddings must be of the weight's type, or of 16 bits beside a float32 weight");
    in.tokens = tokens.contiguous();
    p.tokens = in.tokens.data_ptr();
    p.token_bytes = (int)tokens.element_size();
    if (given(lengths)) {
        TORCH_CHECK(batched, "lengths need tokens [B, L], got ", tokens.sizes());
        check_on(*lengths, tokens, "lengths");
        TORCH_CHECK(lengths->scalar_type() == torch::kInt32 && lengths->dim() == 1 &&
                        lengths->size(0) == p.B,
                    "lengths must be int32 [B] with B = ", p.B, ", got ", lengths->scalar_type(),
                    " ", lengths->sizes());
        in.lengths = lengths->contiguous();
        p.lengths = in.lengths.data_ptr<int>();
    }
    TORCH_CHECK(padding >= -1 && padding < p.V, "padding must be a token of ", p.V,
                ", got ", padding);
    p.padding = padding;
    TORCH_CHECK(std::isfinite(scale) && std::isfinite((float)scale), "scale must be finite, got ",
                scale);
    p.scale = (float)scale;
    return in;
}

int type_of(at::ScalarType t, const char* name) {
    TORCH_CHECK(t == torch::kFloat32 || t == torch::kFloat16 || t == torch::kBFloat16, name,
                " must be float32, float16 or bfloat16, got ", t);
    return t == torch::kFloat32 ? D2P_FLOAT32 : t == torch::kFloat16 ? D2P_FLOAT16 : D2P_BFLOAT16;
}

Tensor token_embedding(const Tensor& tokens, const Tensor& weight, const OptTensor& lengths,
                       double scale, int64_t padding, at::ScalarType dtype) {
    TORCH_CHECK(weight.is_cuda(), "weight must be a CUDA tensor");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(weight.device());
    check_on(tokens, weight, "tokens");
    TORCH_CHECK(weight.dim() == 2, "weight must be 2D (tokens, features), got ", weight.dim(), "D");
    const auto in = embed_inputs(tokens, lengths, scale, padding, weight.size(0), weight.size(1),
                                 type_code(weight, "weight"), type_of(dtype, "dtype"));
    const Tensor w = weight.contiguous();
    auto sizes = tokens.sizes().vec();
    sizes.push_back(weight.size(1));
    Tensor out = torch::empty(sizes, weight.options().dtype(dtype));
    D2P_CALL(d2p_token_embedding(&in.p, w.data_ptr(), out.data_ptr(), current_stream()));
    return out;
}

Tensor token_embedding_backward(const Tensor& grad_, const Tensor& tokens, const OptTensor& lengths,
                                double scale, int64_t padding, int64_t rows, at::ScalarType dtype) {
    TORCH_CHECK(grad_.is_cuda(), "grad must be a CUDA tensor");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(grad_.device());
    check_on(tokens, grad_, "tokens");
    TORCH_CHECK(grad_.dim() == tokens.dim() + 1, "grad must have tokens' shape and features, got ",
                grad_.sizes());
    for (int64_t d = 0; d < tokens.dim(); ++d)
        TORCH_CHECK(grad_.size(d) == tokens.size(d), "grad must have tokens' shape ",
                    tokens.sizes(), " and features, got ", grad_.sizes());
    auto in = embed_inputs(tokens, lengths, scale, padding, rows, grad_.size(-1),
                           type_of(dtype, "dtype"), type_code(grad_, "grad"));
    const Tensor grad = tokens.dim() == 2 ? adjacent_rows(grad_) : grad_.contiguous();
    in.p.grad = tokens.dim() == 2 ? row_strides(grad)
                                  : d2p_row_strides{0, grad.size(-1)};
    Tensor dw = torch::empty({rows, grad.size(-1)}, grad.options().dtype(dtype));
    const size_t bytes = d2p_token_embedding_backward_workspace_bytes(&in.p);
    Tensor ws = workspace(bytes, grad);
    D2P_CALL(d2p_token_embedding_backward(&in.p, grad.data_ptr(), dw.data_ptr(), ws.data_ptr(),
                                          bytes, current_stream()));
    return dw;
}

auto call_embedding(const Tensor& tokens, const Tensor& weight, const OptTensor& lengths,
                    double scale, int64_t padding, at::ScalarType dtype) {
    static auto op = operator_handle<decltype(token_embedding)>("d2p_amd::token_embedding");
    return op.call(tokens, weight, lengths, scale, padding, dtype);
}

class TokenEmbeddingFunction : public torch::autograd::Function<TokenEmbeddingFunction> {
   public:
    static Tensor forward(AutogradContext* ctx, const Tensor& tokens, const Tensor& weight,
                          const OptTensor& lengths, double scale, int64_t padding,
                          at::ScalarType dtype) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({tokens, lengths.value_or(Tensor())});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding;
        ctx->saved_data["rows"] = weight.size(0);
        ctx->saved_data["dtype"] = (int64_t)weight.scalar_type();
        return call_embedding(tokens, weight, lengths, scale, padding, dtype);
    }
    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const auto s = ctx->get_saved_variables();
        no_tangents("token_embedding's backward", {&grads[0]});
        BelowAutograd below;
        static auto op = operator_handle<decltype(token_embedding_backward)>(
            "d2p_amd::token_embedding_backward");
        Tensor dw = op.call(grads[0], s[0], saved(s[1]), ctx->saved_data["scale"].toDouble(),
                            ctx->saved_data["padding"].toInt(), ctx->saved_data["rows"].toInt(),
                            (at::ScalarType)ctx->saved_data["dtype"].toInt());
        return {Tensor(), dw, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor token_embedding_autograd(const Tensor& tokens, const Tensor& weight,
                                const OptTensor& lengths, double scale, int64_t padding,
                                at::ScalarType dtype) {
    no_tangents("token_embedding", {&weight});
    if (differentiates({&weight}))
        return TokenEmbeddingFunction::apply(tokens, weight, lengths, scale, padding, dtype);
    at::AutoDispatchBelowADInplaceOrView below;
    return call_embedding(tokens, weight, lengths, scale, padding, dtype);
}

// ---------------------------------------------------------------------------
// residual stream
// ---------------------------------------------------------------------------
struct ResidualInputs {
    d2p_residual_norm_params p{};
    Tensor weight, bias, post_weight, post_bias, gate;    // as the kernels read them
};

d2p_vector vector_of(const OptTensor& v, const Tensor& x, const char* name, Tensor* keep) {
    if (!given(v)) return {nullptr, D2P_FLOAT32};
    check_on(*v, x, name);
    TORCH_CHECK(v->dim() == 1 && v->size(0) == x.size(2), name, " must be [", x.size(2), "], got ",
                v->sizes());
    const int type = type_code(*v, name);
    *keep = v->contiguous();
    return {keep->data_ptr(), type};
}

void check_3d(const Tensor& t, const Tensor& x, at::ScalarType type, const char* name) {
    check_on(t, x, name);
    TORCH_CHECK(t.sizes() == x.sizes(), name, " must have x's shape ", x.sizes(), ", got ", t.sizes());
    TORCH_CHECK(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
}

// All but x's, y's and their gradients' strides; `dtype`: the block's
ResidualInputs residual_inputs(const Tensor& x, const OptTensor& weight, const OptTensor& bias,
                               const OptTensor& post_weight, const OptTensor& post_bias,
                               const OptTensor& gate, int64_t norm, int64_t post_norm, double scale,
                               double residual_scale, double eps, at::ScalarType dtype) {
    ResidualInputs in;
    auto& p = in.p;
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    TORCH_CHECK(x.dim() == 3, "x must be 3D (batch, length, features), got ", x.dim(), "D");
    p.dtype = type_code(x, "x");
    p.block_dtype = type_of(dtype, "dtype");
    TORCH_CHECK(p.block_dtype == p.dtype || p.dtype == D2P_FLOAT32,
                "the block's type must be x's, or 16 bits beside a float32 x, got ", dtype, " and ",
                x.scalar_type());
    p.B = dim32(x.size(0), "batch size");
    p.L = dim32(x.size(1), "length");
    TORCH_CHECK(x.size(2) >= 8 && x.size(2) <= 8192, "features must be between 8 and 8192, got ",
                x.size(2));
    p.D = (int)x.size(2);
    TORCH_CHECK((int64_t)p.B * p.L < int64_t(1) << 31, "too many rows: ", x.sizes());
    p.norm = (int)norm;
    p.post_norm = (int)post_norm;
    p.weight = vector_of(weight, x, "weight", &in.weight);
    p.bias = vector_of(bias, x, "bias", &in.bias);
    p.post_weight = vector_of(post_weight, x, "post_weight", &in.post_weight);
    p.post_bias = vector_of(post_bias, x, "post_bias", &in.post_bias);
    if (given(gate)) {
        check_on(*gate, x, "gate");
        p.gate_dtype = type_code(*gate, "gate");
        TORCH_CHECK(p.gate_dtype == D2P_FLOAT32 || p.gate_dtype == p.block_dtype,
                    "gate must be float32 or of the block's type ", dtype, ", got ",
                    gate->scalar_type());
        const bool rows = gate->dim() == 3 && gate->size(0) == x.size(0) && gate->size(2) == x.size(2);
        if (gate->dim() == 1 && gate->size(0) == x.size(2)) p.gate_kind = D2P_GATE_FEATURE;
        else if (rows && gate->size(1) == x.size(1)) p.gate_kind = D2P_GATE_TOKEN;
        else if (rows && gate->size(1) == 1) p.gate_kind = D2P_GATE_SEQUENCE;
        else
            TORCH_CHECK(false, "gate must be [D], [B, 1, D] or [B, L, D] beside x ", x.sizes(),
                        ", got ", gate->sizes());
        in.gate = p.gate_kind == D2P_GATE_FEATURE ? gate->contiguous() : adjacent_rows(*gate);
        p.gate = in.gate.data_ptr();
        if (p.gate_kind != D2P_GATE_FEATURE) p.gate_strides = row_strides(in.gate);
    }
    TORCH_CHECK(std::isfinite((float)scale) && std::isfinite((float)residual_scale),
                "scale and residual_scale must be finite, got ", scale, " and ", residual_scale);
    p.scale = (float)scale;
    p.residual_scale = (float)residual_scale;
    TORCH_CHECK(eps >= 0 && std::isfinite((float)eps), "eps must not be negative, got ", eps);
    p.eps = (float)eps;
    return in;
}

using ThreeTensors = std::tuple<Tensor, Tensor, Tensor>;

ThreeTensors residual_norm_forward(const Tensor& x_, const OptTensor& y_, const OptTensor& weight,
                                   const OptTensor& bias, const OptTensor& post_weight,
                                   const OptTensor& post_bias, const OptTensor& gate, int64_t norm,
                                   int64_t post_norm, double scale, double residual_scale,
                                   double eps, at::ScalarType dtype, bool stats) {
    TORCH_CHECK(x_.is_cuda(), "x must be a CUDA tensor");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(x_.device());
    auto in = residual_inputs(x_, weight, bias, post_weight, post_bias, gate, norm, post_norm,
                              scale, residual_scale, eps, dtype);
    const bool block = given(y_);
    if (block) check_3d(*y_, x_, dtype, "y");
    const Tensor x = adjacent_rows(x_), y = block ? adjacent_rows(*y_) : Tensor();
    in.p.x = row_strides(x);
    if (block) in.p.y = row_strides(y);
    in.p.with_y = block;
    Tensor h = block ? torch::empty(x.sizes(), x.options()) : Tensor();
    Tensor n = norm ? torch::empty(x.sizes(), x.options().dtype(dtype)) : Tensor();
    Tensor st = stats ? torch::empty({x.size(0), x.size(1), 4}, x.options().dtype(torch::kFloat32))
                      : Tensor();
    D2P_CALL(d2p_residual_norm(&in.p, x.data_ptr(), block ? y.data_ptr() : nullptr,
                               block ? h.data_ptr() : nullptr, norm ? n.data_ptr() : nullptr,
                               stats ? st.data_ptr<float>() : nullptr, current_stream()));
    return {h, n, st};
}

using SevenTensors = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;

// h: the forward's for float32, x for 16 bits and where there is no y; needed with dn.  stats: needed
// with a norm.  dy comes back undefined where it equals dx, and so does every gradient that `wanted`
// (bits: gate, then the four vectors) leaves out.
SevenTensors residual_norm_backward(const OptTensor& dh_, const OptTensor& dn_, const OptTensor& h_,
                                    const OptTensor& y_, const OptTensor& stats,
                                    const OptTensor& weight, const OptTensor& bias,
                                    const OptTensor& post_weight, const OptTensor& post_bias,
                                    const OptTensor& gate, int64_t norm, int64_t post_norm,
                                    double scale, double residual_scale, double eps,
                                    at::ScalarType dtype, bool block, int64_t wanted) {
    TORCH_CHECK(given(h_) || (given(dh_) && !(given(dn_) && norm)), "h is needed");
    const Tensor& like = given(h_) ? *h_ : *dh_;    // of x's sizes and type
    TORCH_CHECK(like.is_cuda(), "h must be a CUDA tensor");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(like.device());
    auto in = residual_inputs(like, weight, bias, post_weight, post_bias, gate, norm, post_norm,
                              scale, residual_scale, eps, dtype);
    in.p.with_y = block;
    Tensor h, dh, dn, y;
    if (given(h_)) {
        h = block && h_->scalar_type() == torch::kFloat32 ? h_->contiguous() : adjacent_rows(*h_);
        in.p.x = row_strides(h);
    }
    if (given(dh_)) {
        check_3d(*dh_, like, like.scalar_type(), "grad of h");
        dh = adjacent_rows(*dh_);
        in.p.dh = row_strides(dh);
    }
    if (given(dn_) && norm) {
        check_3d(*dn_, like, dtype, "grad of n");
        dn = adjacent_rows(*dn_);
        in.p.dn = row_strides(dn);
    }
    if (given(y_)) {
        check_3d(*y_, like, dtype, "y");
        y = adjacent_rows(*y_);
        in.p.y = row_strides(y);
    }
    if (given(stats)) {
        check_on(*stats, like, "stats");
        TORCH_CHECK(stats->scalar_type() == torch::kFloat32 && stats->is_contiguous() &&
                        stats->numel() == 4 * like.size(0) * like.size(1),
                    "stats must be float32 [B, L, 4], got ", stats->sizes());
    }
    const bool same = block && !post_norm && !given(gate) && scale == residual_scale &&
                      like.scalar_type() == dtype;
    Tensor dx = torch::empty(like.sizes(), like.options());
    Tensor dy = block && !same ? torch::empty(like.sizes(), like.options().dtype(dtype)) : Tensor();
    auto of = [&](const OptTensor& v, int bit) {
        return given(v) && (wanted >> bit & 1) ? torch::empty(v->sizes(), v->options()) : Tensor();
    };
    Tensor dgate = of(gate, 0), dw = of(weight, 1), db = of(bias, 2), dpw = of(post_weight, 3),
           dpb = of(post_bias, 4);
    auto data = [](const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; };
    const size_t bytes = d2p_residual_norm_backward_workspace_bytes(&in.p);
    Tensor ws = workspace(bytes, like);
    D2P_CALL(d2p_residual_norm_backward(&in.p, data(dh), data(dn), data(h), data(y),
                                        given(stats) ? stats->data_ptr<float>() : nullptr,
                                        dx.data_ptr(), data(dy), data(dgate), data(dw), data(db),
                                        data(dpw), data(dpb), ws.data_ptr(), bytes,
                                        current_stream()));
    return {dx, dy, dgate, dw, db, dpw, dpb};
}

auto call_residual(const Tensor& x, const OptTensor& y, const OptTensor& weight,
                   const OptTensor& bias, const OptTensor& post_weight, const OptTensor& post_bias,
                   const OptTensor& gate, int64_t norm, int64_t post_norm, double scale,
                   double residual_scale, double eps, at::ScalarType dtype, bool stats) {
    static auto op =
        operator_handle<decltype(residual_norm_forward)>("d2p_amd::residual_norm_forward");
    return op.call(x, y, weight, bias, post_weight, post_bias, gate, norm, post_norm, scale,
                   residual_scale, eps, dtype, stats);
}

class ResidualNormFunction : public torch::autograd::Function<ResidualNormFunction> {
   public:
    static tensor_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& y,
                               const OptTensor& weight, const OptTensor& bias,
                               const OptTensor& post_weight, const OptTensor& post_bias,
                               const OptTensor& gate, int64_t norm, int64_t post_norm, double scale,
                               double residual_scale, double eps, at::ScalarType dtype) {
        at::AutoDispatchBelowADInplaceOrView below;
        Tensor h, n, stats;
        std::tie(h, n, stats) =
            call_residual(x, y, weight, bias, post_weight, post_bias, gate, norm, post_norm, scale,
                          residual_scale, eps, dtype, norm || post_norm);
        auto wants = [](const OptTensor& t) { return given(t) && t->requires_grad(); };
        // y enters the gradients through its own norm, the gate's, and h where that is rounded; h
        // through its norm
        const bool wide = x.scalar_type() == torch::kFloat32;
        const bool keep_y = post_norm || wants(gate) || (norm && !wide);
        ctx->save_for_backward({!norm ? Tensor() : given(y) && wide ? h : x,
                                keep_y ? y.value_or(Tensor()) : Tensor(), stats,
                                weight.value_or(Tensor()), bias.value_or(Tensor()),
                                post_weight.value_or(Tensor()), post_bias.value_or(Tensor()),
                                gate.value_or(Tensor())});
        ctx->saved_data["norm"] = norm;
        ctx->saved_data["post_norm"] = post_norm;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["residual_scale"] = residual_scale;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["dtype"] = (int64_t)dtype;
        ctx->saved_data["block"] = given(y);
        ctx->saved_data["wanted"] = int64_t(wants(gate)) | wants(weight) << 1 | wants(bias) << 2 |
                                    wants(post_weight) << 3 | wants(post_bias) << 4;
        ctx->set_materialize_grads(false);
        // (a function's results are tensors; residual_norm_autograd leaves these out)
        for (Tensor* t : {&h, &n})
            if (!t->defined()) *t = torch::empty({0}, x.options());
        return {h, n};
    }
    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const auto s = ctx->get_saved_variables();
        auto& d = ctx->saved_data;
        no_tangents("residual_norm's backward", {&grads[0], &grads[1]});
        tensor_list out(13);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        BelowAutograd below;
        static auto op =
            operator_handle<decltype(residual_norm_backward)>("d2p_amd::residual_norm_backward");
        const bool block = d["block"].toBool();
        const int64_t wanted = d["wanted"].toInt();
        auto [dx, dy, dgate, dw, db, dpw, dpb] =
            op.call(saved(grads[0]), saved(grads[1]), saved(s[0]), saved(s[1]), saved(s[2]),
                    saved(s[3]), saved(s[4]), saved(s[5]), saved(s[6]), saved(s[7]), d["norm"].toInt(),
                    d["post_norm"].toInt(), d["scale"].toDouble(), d["residual_scale"].toDouble(),
                    d["eps"].toDouble(), (at::ScalarType)d["dtype"].toInt(), block, wanted);
        out[0] = dx;
        if (block) out[1] = dy.defined() ? dy : dx;
        out[2] = dw;
        out[3] = db;
        out[4] = dpw;
        out[5] = dpb;
        out[6] = dgate;
        return out;
    }
};

std::tuple<Tensor, Tensor> residual_norm(const Tensor& x, const OptTensor& y,
                                         const OptTensor& weight, const OptTensor& bias,
                                         const OptTensor& post_weight, const OptTensor& post_bias,
                                         const OptTensor& gate, int64_t norm, int64_t post_norm,
                                         double scale, double residual_scale, double eps,
                                         at::ScalarType dtype) {
    auto [h, n, stats] = residual_norm_forward(x, y, weight, bias, post_weight, post_bias, gate,
                                               norm, post_norm, scale, residual_scale, eps, dtype,
                                               false);
    return {h, n};
}

std::tuple<Tensor, Tensor> residual_norm_autograd(
    const Tensor& x, const OptTensor& y, const OptTensor& weight, const OptTensor& bias,
    const OptTensor& post_weight, const OptTensor& post_bias, const OptTensor& gate, int64_t norm,
    int64_t post_norm, double scale, double residual_scale, double eps, at::ScalarType dtype) {
    const Tensor t[] = {y.value_or(Tensor()),         weight.value_or(Tensor()),
                        bias.value_or(Tensor()),      post_weight.value_or(Tensor()),
                        post_bias.value_or(Tensor()), gate.value_or(Tensor())};
    no_tangents("residual_norm", {&x, &t[0], &t[1], &t[2], &t[3], &t[4], &t[5]});
    if (differentiates({&x, &t[0], &t[1], &t[2], &t[3], &t[4], &t[5]})) {
        auto r = ResidualNormFunction::apply(x, y, weight, bias, post_weight, post_bias, gate, norm,
                                             post_norm, scale, residual_scale, eps, dtype);
        return {given(y) ? r[0] : Tensor(), norm ? r[1] : Tensor()};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    auto [h, n, stats] = call_residual(x, y, weight, bias, post_weight, post_bias, gate, norm,
                                       post_norm, scale, residual_scale, eps, dtype, false);
    return {h, n};
}

// ---------------------------------------------------------------------------
// gradient norm and clipping
// ---------------------------------------------------------------------------

// The list as the kernels take it: memory in any dense order is numbers after numbers; other
// tensors are copied (and kept in `copies`).
std::vector<d2p_tensor> tensor_list_of(at::TensorList ts, std::vector<Tensor>& copies) {
    std::vector<d2p_tensor> list;
    list.reserve(ts.size());
    for (const Tensor& t : ts) {
        check_on(t, ts[0], "every tensor");
        const int type = type_code(t, "every tensor");
        const Tensor* from = &t;
        if (!t.is_non_overlapping_and_dense()) {
            copies.push_back(t.contiguous());
            from = &copies.back();
        }
        list.push_back({from->data_ptr(), nullptr, from->numel(), type});
    }
    return list;
}

Tensor global_norm(at::TensorList ts) {
    TORCH_CHECK(!ts.empty(), "need at least one tensor");
    TORCH_CHECK(ts[0].is_cuda(), "every tensor must be a CUDA tensor");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(ts[0].device());
    std::vector<Tensor> copies;
    copies.reserve(ts.size());
    const auto list = tensor_list_of(ts, copies);
    Tensor norm = torch::empty({}, ts[0].options().dtype(torch::kFloat32));
    const size_t bytes = d2p_global_norm_workspace_bytes((int)list.size());
    Tensor ws = workspace(bytes, ts[0]);
    D2P_CALL(d2p_global_norm(list.data(), (int)list.size(), norm.data_ptr<float>(), ws.data_ptr(),
                             bytes, current_stream()));
    return norm;
}

Tensor clip_lists(std::vector<d2p_tensor>& list, const Tensor& like, double max_norm) {
    TORCH_CHECK(max_norm >= 0, "max_norm must not be negative, got ", max_norm);
    Tensor norm = torch::empty({}, like.options().dtype(torch::kFloat32));
    const size_t bytes = d2p_global_norm_workspace_bytes((int)list.size());
    Tensor ws = workspace(bytes, like);
    D2P_CALL(d2p_clip_by_norm(list.data(), (int)list.size(), max_norm, norm.data_ptr<float>(),
                              ws.data_ptr(), bytes, current_stream()));
    return norm;
}

// Contiguous memory for results, or, for a dense source, memory in its order.  One allocation
// holds them all, each at a multiple of 256 bytes: one apiece takes the host a microsecond each.
std::vector<Tensor> results_for(at::TensorList ts, std::vector<d2p_tensor>& list) {
    int64_t bytes = 0;
    for (const auto& t : list) bytes += (t.n * (t.dtype == D2P_FLOAT32 ? 4 : 2) + 255) / 256 * 256;
    Tensor all = workspace(bytes, ts[0]);
    std::vector<Tensor> out;
    out.reserve(ts.size());
    int64_t at = 0;
    for (size_t i = 0; i < ts.size(); ++i) {
        const Tensor& t = ts[i];
        const int64_t size = t.element_size();
        auto r = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()),
                                                          all.key_set(), t.dtype());
        auto* impl = r.unsafeGetTensorImpl();
        if (t.is_non_overlapping_and_dense()) {
            impl->set_sizes_and_strides(t.sizes(), t.strides(), at / size);
        } else {
            impl->set_storage_offset(at / size);
            impl->set_sizes_contiguous(t.sizes());
        }
        list[i].dst = (char*)all.data_ptr() + at;
        at += (list[i].n * size + 255) / 256 * 256;
        out.push_back(std::move(r));
    }
    return out;
}

std::tuple<std::vector<Tensor>, Tensor> clip_gradients(at::TensorList ts, double max_norm) {
    TORCH_CHECK(!ts.empty(), "need at least one tensor");
    TORCH_CHECK(ts[0].is_cuda(), "every tensor must be a CUDA tensor");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(ts[0].device());
    std::vector<Tensor> copies;
    copies.reserve(ts.size());
    auto list = tensor_list_of(ts, copies);
    std::vector<Tensor> out = results_for(ts, list);
    Tensor norm = clip_lists(list, ts[0], max_norm);
    return {std::move(out), norm};
}

// Results that share memory with each other, or with a source other than their own, would be
// read after they are written.  `more`: results that are written later, from memory of their own.
void check_apart(const std::vector<d2p_tensor>& list, const std::vector<d2p_tensor>& more) {
    using Range = std::pair<uintptr_t, uintptr_t>;
    auto range = [](const void* from, const d2p_tensor& t) {
        return Range((uintptr_t)from, (uintptr_t)from + t.n * (t.dtype == D2P_FLOAT32 ? 4 : 2));
    };
    std::vector<Range> results;
    results.reserve(list.size());
    for (const auto& t : list)
        if (t.n) results.push_back(range(t.dst, t));
    if (!std::is_sorted(results.begin(), results.end())) std::sort(results.begin(), results.end());
    bool apart = true;
    for (size_t i = 1; i < results.size(); ++i) apart &= results[i - 1].second <= results[i].first;
    for (const auto& t : list) {
        if (!t.n || t.src == t.dst) continue;
        const Range r = range(t.src, t);
        // the first result that ends after the source begins
        auto it = std::upper_bound(results.begin(), results.end(), r.first,
                                   [](uintptr_t x, const Range& y) { return x < y.second; });
        apart &= it == results.end() || it->first >= r.second;
    }
    if (!more.empty()) {        // (the sources have all been read by then)
        for (const auto& t : more)
            if (t.n) results.push_back(range(t.dst, t));
        std::sort(results.begin(), results.end());
        for (size_t i = 1; i < results.size(); ++i) apart &= results[i - 1].second <= results[i].first;
    }
    TORCH_CHECK(apart, "tensors share memory that a result is written to");
}

Tensor clip_gradients_into(at::TensorList ts, double max_norm, at::TensorList out) {
    TORCH_CHECK(!ts.empty(), "need at least one tensor");
    TORCH_CHECK(ts[0].is_cuda(), "every tensor must be a CUDA tensor");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(ts[0].device());
    TORCH_CHECK(out.size() == ts.size(), "out must have ", ts.size(), " tensors, got ", out.size());
    std::vector<Tensor> copies;
    copies.reserve(ts.size());
    auto list = tensor_list_of(ts, copies);
    // results in another order than their source's, or in no dense memory; those that are dense
    std::vector<std::pair<size_t, Tensor>> late;
    std::vector<d2p_tensor> late_dense;
    for (size_t i = 0; i < list.size(); ++i) {
        check_on(out[i], ts[0], "every tensor of out");
        TORCH_CHECK(out[i].sizes() == ts[i].sizes() && out[i].scalar_type() == ts[i].scalar_type(),
                    "out must have the tensors' shapes and types, got ", out[i].sizes(), " ",
                    out[i].scalar_type(), " for ", ts[i].sizes(), " ", ts[i].scalar_type());
        const bool dense = ts[i].is_non_overlapping_and_dense();
        if (dense ? out[i].strides() == ts[i].strides() : out[i].is_contiguous()) {
            list[i].dst = out[i].data_ptr();
        } else {
            if (list[i].n) at::assert_no_internal_overlap(out[i]);
            if (out[i].is_non_overlapping_and_dense())
                late_dense.push_back({nullptr, out[i].data_ptr(), list[i].n, list[i].dtype});
            late.emplace_back(i, dense ? torch::empty_strided(ts[i].sizes(), ts[i].strides(),
                                                              ts[i].options())
                                       : torch::empty(ts[i].sizes(), ts[i].options()));
            list[i].dst = late.back().second.data_ptr();
        }
    }
    check_apart(list, late_dense);
    Tensor norm = clip_lists(list, ts[0], max_norm);
    for (auto& [i, t] : late) out[i].copy_(t);
    return norm;
}

void check_undifferentiated(at::TensorList ts, const char* name) {
    for (const Tensor& t : ts) {
        if (!t.unsafeGetTensorImpl()->autograd_meta()) continue;    // of no graph
        no_tangents(name, {&t});
        TORCH_CHECK_NOT_IMPLEMENTED(!differentiates({&t}), name,
                                    " has no derivative; call it under torch.no_grad()");
    }
}

Tensor global_norm_autograd(at::TensorList ts) {
    check_undifferentiated(ts, "global_norm");
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = operator_handle<decltype(global_norm)>("d2p_amd::global_norm");
    return op.call(ts);
}
std::tuple<std::vector<Tensor>, Tensor> clip_gradients_autograd(at::TensorList ts, double max_norm) {
    check_undifferentiated(ts, "clip_gradients");
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = operator_handle<decltype(clip_gradients)>("d2p_amd::clip_gradients");
    return op.call(ts, max_norm);
}
Tensor clip_gradients_into_autograd(at::TensorList ts, double max_norm, at::TensorList out) {
    check_undifferentiated(ts, "clip_gradients");
    check_undifferentiated(out, "clip_gradients");
    for (const Tensor& t : out)
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = operator_handle<decltype(clip_gradients_into)>("d2p_amd::clip_gradients_into");
    return op.call(ts, max_norm, out);
}

}  // namespace

#define RESIDUAL_VECTORS                                                                     \
    "Tensor? weight, Tensor? bias, Tensor? post_weight, Tensor? post_bias, Tensor? gate, "
#define RESIDUAL_OPTIONS                                                                     \
    "int norm, int post_norm, float scale, float residual_scale, float eps, ScalarType dtype"

TORCH_LIBRARY_FRAGMENT(d2p_amd, m) {
    m.def("token_embedding(Tensor tokens, Tensor weight, Tensor? lengths, float scale, "
          "int padding, ScalarType dtype) -> Tensor");
    m.def("token_embedding_backward(Tensor grad, Tensor tokens, Tensor? lengths, float scale, "
          "int padding, int rows, ScalarType dtype) -> Tensor");
    m.def("residual_norm(Tensor x, Tensor? y, " RESIDUAL_VECTORS RESIDUAL_OPTIONS
          ") -> (Tensor, Tensor)");
    m.def("residual_norm_forward(Tensor x, Tensor? y, " RESIDUAL_VECTORS RESIDUAL_OPTIONS
          ", bool stats) -> (Tensor, Tensor, Tensor)");
    m.def("residual_norm_backward(Tensor? dh, Tensor? dn, Tensor? h, Tensor? y, Tensor? stats, "
          RESIDUAL_VECTORS RESIDUAL_OPTIONS ", bool block, int wanted) -> "
          "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("global_norm(Tensor[] tensors) -> Tensor");
    m.def("clip_gradients(Tensor[] tensors, float max_norm) -> (Tensor[], Tensor)");
    m.def("clip_gradients_into(Tensor[] tensors, float max_norm, Tensor(a!)[] out) -> Tensor");
}

TORCH_LIBRARY_IMPL(d2p_amd, CUDA, m) {
    m.impl("token_embedding", token_embedding);
    m.impl("token_embedding_backward", token_embedding_backward);
    m.impl("residual_norm", residual_norm);
    m.impl("residual_norm_forward", residual_norm_forward);
    m.impl("residual_norm_backward", residual_norm_backward);
    m.impl("global_norm", global_norm);
    m.impl("clip_gradients", clip_gradients);
    m.impl("clip_gradients_into", clip_gradients_into);
}

TORCH_LIBRARY_IMPL(d2p_amd, Autograd, m) {
    m.impl("token_embedding", token_embedding_autograd);
    m.impl("residual_norm", residual_norm_autograd);
    m.impl("global_norm", global_norm_autograd);
    m.impl("clip_gradients", clip_gradients_autograd);
    m.impl("clip_gradients_into", clip_gradients_into_autograd);
    for (const char* name : {"token_embedding_backward", "residual_norm_forward",
                             "residual_norm_backward"})
        m.impl(name, torch::autograd::autogradNotImplementedFallback());
}

TORCH_LIBRARY_IMPL(d2p_amd, CPU, m) {
    for (const char* name :
         {"token_embedding", "token_embedding_backward", "residual_norm", "residual_norm_forward",
          "residual_norm_backward", "global_norm", "clip_gradients", "clip_gradients_into"})
        m.impl(name, torch::CppFunction::makeFromBoxedFunction<&cpu_boxed>());
}
