// PyTorch bindings of the operators round the experts that need no Buffer: residual and norm (also with rows in 8 bits), routing, rows
// grouped by expert and brought back, with their gradients.
// Schemas are added to the library that bindings.cpp defines.
#include "bindings_common.h"
#include "runtime/layer_ops.h"

namespace {

using namespace umdk;

using Two = std::tuple<at::Tensor, at::Tensor>;
using Three = std::tuple<at::Tensor, at::Tensor, at::Tensor>;
using Four = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

cudaStream_t stream_now() { return at::cuda::getCurrentCUDAStream().stream(); }
void* data_or_null(const at::Tensor& t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }
float* floats_or_null(const at::Tensor& t) { return static_cast<float*>(data_or_null(t)); }
at::Tensor none_of(const at::Tensor& like) { return at::empty({0}, like.options()); }
at::Tensor cuda_like(const at::Tensor& t) { return cuda_empty(t.sizes(), t.scalar_type(), t); }
at::Tensor cuda_none(const at::Tensor& like) { return cuda_empty({0}, like.scalar_type(), like); }

// ------------------------------------------------------------------------------------------------
// Norm
// ------------------------------------------------------------------------------------------------
struct NormProblem {
    int64_t rows;
    int h, dtype, res_type, weight_type;
};

NormProblem check_norm(const char* op, const at::Tensor& x, const OptTensor& residual, const at::Tensor& weight, double eps) {
    check_operand(x, x, "x");
    check_operand(weight, x, "weight");
    NormProblem p{};
    p.dtype = dtype_of(x.scalar_type(), "x");
    CAM_ASSERT(x.dim() >= 1 && x.size(-1) >= 1, op, ": x must be [..., h]");
    const int64_t h = x.size(-1);
    CAM_ASSERT(h <= 16384, op, ": rows of ", num(h), " values; at most 16384");
    CAM_ASSERT(weight.dim() == 1 && weight.size(0) == h && (weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat), op,
               ": weight must be [", num(h), "] of x's type or float32");
    CAM_ASSERT(eps >= 0.0, op, ": eps must not be negative");
    p.weight_type = dtype_of(weight.scalar_type(), "weight");
    p.res_type = p.dtype;
    if (given(residual)) {
        check_operand(*residual, x, "residual");
        CAM_ASSERT(residual->sizes() == x.sizes() && (residual->scalar_type() == x.scalar_type() || residual->scalar_type() == at::kFloat), op,
                   ": residual must be ", shape(x.sizes()), " of x's type or float32");
        p.res_type = dtype_of(residual->scalar_type(), "residual");
    }
    p.h = static_cast<int>(h);
    p.rows = x.numel() / h;
    CAM_ASSERT(p.rows < (1ll << 31) - 512, op, ": ", num(p.rows), " rows");
    return p;
}

// y, sum (undefined without a residual), rstd (undefined unless kept)
Three norm_forward(const char* op, const at::Tensor& x, const OptTensor& residual, const at::Tensor& weight, double eps, bool keep) {
    const NormProblem p = check_norm(op, x, residual, weight, eps);
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor y = cuda_like(x), sum, rstd;
    if (given(residual)) sum = cuda_like(*residual);
    if (keep) rstd = cuda_empty({p.rows}, at::kFloat, x);
    if (p.rows == 0) return {y, sum, rstd};
    CAM_RT(cam_rms_norm(x.data_ptr(), p.dtype, given(residual) ? residual->data_ptr() : nullptr, p.res_type, weight.data_ptr(), p.weight_type, p.rows,
                        p.h, static_cast<float>(eps), y.data_ptr(), data_or_null(sum), floats_or_null(rstd), 0, nullptr, nullptr, stream_now()));
    return {y, sum, rstd};
}

at::Tensor rms_norm_cuda(const at::Tensor& x, const at::Tensor& weight, double eps) {
    return std::get<0>(norm_forward("rms_norm", x, c10::nullopt, weight, eps, false));
}
Two add_rms_norm_cuda(const at::Tensor& x, const at::Tensor& residual, const at::Tensor& weight, double eps) {
    auto [y, sum, rstd] = norm_forward("add_rms_norm", x, residual, weight, eps, false);
    return {y, sum};
}
Three rms_norm_train_cuda(const at::Tensor& x, const OptTensor& residual, const at::Tensor& weight, double eps) {
    auto out = norm_forward("rms_norm_train", x, residual, weight, eps, true);
    if (!std::get<1>(out).defined()) std::get<1>(out) = cuda_none(x);
    return out;
}

// dx (of dy's type), dresidual (of the sum's type, empty where that is dx's: then they are the same numbers), dweight
template <class Like, class None>
Three norm_grads_empty(Like like, None none, const at::Tensor& dy, const at::Tensor& sum, const at::Tensor& weight, bool need_dx, bool need_dres, bool need_dw) {
    const bool one = dy.scalar_type() == sum.scalar_type();
    return {need_dx || (one && need_dres) ? like(dy) : none(dy), !one && need_dres ? like(sum) : none(sum), need_dw ? like(weight) : none(weight)};
}

Three rms_norm_backward_cuda(const at::Tensor& dy, const OptTensor& dsum, const at::Tensor& sum, const at::Tensor& weight, const at::Tensor& rstd,
                             bool need_dx, bool need_dres, bool need_dw) {
    const NormProblem p = check_norm("rms_norm_backward", dy, sum, weight, 0.0);
    check_operand(rstd, dy, "rstd");
    CAM_ASSERT(rstd.scalar_type() == at::kFloat && rstd.numel() == p.rows, "rms_norm_backward: rstd must be float32 with one value per row");
    if (given(dsum)) {
        check_operand(*dsum, dy, "dsum");
        CAM_ASSERT(dsum->sizes() == sum.sizes() && dsum->scalar_type() == sum.scalar_type(), "rms_norm_backward: dsum must be like sum");
    }
    c10::cuda::CUDAGuard guard(dy.device());
    auto out = norm_grads_empty(cuda_like, cuda_none, dy, sum, weight, need_dx, need_dres, need_dw);
    auto& [dx, dres, dw] = out;
    if (p.rows == 0) {
        dw.zero_();
        return out;
    }
    const int parts = cam_rms_norm_backward_parts(p.rows, p.h);
    at::Tensor partial = need_dw ? cuda_empty({parts, p.h}, at::kFloat, dy) : at::Tensor();
    CAM_RT(cam_rms_norm_backward(dy.data_ptr(), p.dtype, given(dsum) ? dsum->data_ptr() : nullptr, sum.data_ptr(), p.res_type, weight.data_ptr(),
                                 p.weight_type, rstd.data_ptr<float>(), p.rows, p.h, data_or_null(dx), data_or_null(dres), data_or_null(dw),
                                 floats_or_null(partial), parts, stream_now()));
    return out;
}

at::ScalarType norm_quant_type(int64_t quant_mode) {
    CAM_ASSERT(quant_mode >= 2 && quant_mode <= 4, "rms_norm_quant: quant_mode must be 2 (int8), 3 (e4m3) or 4 (e4m3, power-of-two scales), got ", num(quant_mode));
    return quant_mode == 2 ? at::kChar : at::kFloat8_e4m3fn;
}

Four rms_norm_quant_cuda(const at::Tensor& x, const at::Tensor& weight, int64_t quant_mode, const OptTensor& residual, double eps, bool with_rows) {
    const NormProblem p = check_norm("rms_norm_quant", x, residual, weight, eps);
    const at::ScalarType qt = norm_quant_type(quant_mode);
    CAM_ASSERT(quant_mode == 2 || p.h % 128 == 0, "rms_norm_quant: e4m3 rows must be a multiple of 128 values, not ", num(p.h));
    c10::cuda::CUDAGuard guard(x.device());
    auto scales_of = x.sizes().vec();
    if (quant_mode == 2) scales_of.pop_back();
    else scales_of.back() = p.h / 128;
    at::Tensor q = cuda_empty(x.sizes(), qt, x), s = cuda_empty(scales_of, at::kFloat, x);
    at::Tensor sum = given(residual) ? cuda_like(*residual) : cuda_none(x), y = with_rows ? cuda_like(x) : cuda_none(x);
    if (p.rows == 0) return {q, s, sum, y};
    CAM_RT(cam_rms_norm(x.data_ptr(), p.dtype, given(residual) ? residual->data_ptr() : nullptr, p.res_type, weight.data_ptr(), p.weight_type, p.rows,
                        p.h, static_cast<float>(eps), data_or_null(y), data_or_null(sum), nullptr, static_cast<int>(quant_mode), q.data_ptr(),
                        s.data_ptr<float>(), stream_now()));
    return {q, s, sum, y};
}

// ------------------------------------------------------------------------------------------------
// Routing
// ------------------------------------------------------------------------------------------------
bool sigmoid_of(c10::string_view score) {
    CAM_ASSERT(score == "softmax" || score == "sigmoid", "moe_route: score must be 'softmax' or 'sigmoid', got '", std::string(score.data(), score.size()), "'");
    return score == "sigmoid";
}

void check_logits(const char* op, const at::Tensor& logits, int64_t k) {
    check_operand(logits, logits, "logits");
    CAM_ASSERT(logits.dim() == 2, op, ": logits must be [T, E]");
    CAM_ASSERT(k >= 1 && k <= 32 && k <= logits.size(1), op, ": k ", num(k), " outside [1, min(", num(logits.size(1)), " experts, 32)]");
    CAM_ASSERT(logits.size(1) <= 1024 && logits.size(0) < (1ll << 31) - 512, op, ": logits ", shape(logits.sizes()), "; at most 1024 experts");
}

Two moe_route_cuda(const at::Tensor& logits, int64_t k, const OptTensor& bias, c10::string_view score, int64_t num_groups, int64_t topk_groups,
                   int64_t group_top, bool renormalize, double scale) {
    check_logits("moe_route", logits, k);
    const bool sigmoid = sigmoid_of(score);
    const int dt = dtype_of(logits.scalar_type(), "logits");
    const int64_t t = logits.size(0), e = logits.size(1);
    if (given(bias)) {
        check_operand(*bias, logits, "bias");
        CAM_ASSERT(bias->scalar_type() == at::kFloat && bias->dim() == 1 && bias->size(0) == e, "moe_route: bias must be float32 [", num(e), "]");
    }
    CAM_ASSERT(num_groups >= 1 && num_groups <= 32 && e % num_groups == 0, "moe_route: ", num(e), " experts in ", num(num_groups), " groups; at most 32 groups of equal size");
    CAM_ASSERT(topk_groups >= 1 && topk_groups <= num_groups, "moe_route: topk_groups ", num(topk_groups), " outside [1, ", num(num_groups), "]");
    CAM_ASSERT(k <= e / num_groups * topk_groups, "moe_route: k ", num(k), " of the ", num(e / num_groups * topk_groups), " experts in ", num(topk_groups), " groups");
    CAM_ASSERT(group_top == 1 || group_top == 2, "moe_route: group_top must be 1 or 2, got ", num(group_top));
    c10::cuda::CUDAGuard guard(logits.device());
    at::Tensor idx = cuda_empty({t, k}, at::kLong, logits), w = cuda_empty({t, k}, at::kFloat, logits);
    if (t == 0) return {idx, w};
    CAM_RT(cam_moe_route(logits.data_ptr(), dt, t, static_cast<int>(e), static_cast<int>(k), given(bias) ? bias->data_ptr<float>() : nullptr, sigmoid,
                         static_cast<int>(num_groups), static_cast<int>(topk_groups), static_cast<int>(group_top), renormalize,
                         static_cast<float>(scale), idx.data_ptr<int64_t>(), w.data_ptr<float>(), stream_now()));
    return {idx, w};
}

at::Tensor moe_route_backward_cuda(const at::Tensor& dweights, const at::Tensor& logits, const at::Tensor& topk_idx, c10::string_view score,
                                   bool renormalize, double scale) {
    CAM_ASSERT(topk_idx.dim() == 2, "moe_route_backward: topk_idx must be int64 [T, k]");
    const int64_t k = topk_idx.size(1);
    check_logits("moe_route_backward", logits, k);
    check_operand(dweights, logits, "dweights");
    check_operand(topk_idx, logits, "topk_idx");
    CAM_ASSERT(topk_idx.scalar_type() == at::kLong && topk_idx.size(0) == logits.size(0), "moe_route_backward: topk_idx must be int64 [T, k]");
    CAM_ASSERT(dweights.scalar_type() == at::kFloat && dweights.sizes() == topk_idx.sizes(), "moe_route_backward: dweights must be float32 [T, k]");
    const int dt = dtype_of(logits.scalar_type(), "logits");
    const bool sigmoid = sigmoid_of(score);
    c10::cuda::CUDAGuard guard(logits.device());
    at::Tensor dlogits = cuda_like(logits);
    if (logits.size(0) == 0) return dlogits;
    CAM_RT(cam_moe_route_backward(dweights.data_ptr<float>(), logits.data_ptr(), dt, topk_idx.data_ptr<int64_t>(), logits.size(0),
                                  static_cast<int>(logits.size(1)), static_cast<int>(k), sigmoid, renormalize, static_cast<float>(scale),
                                  dlogits.data_ptr(), stream_now()));
    return dlogits;
}

// ------------------------------------------------------------------------------------------------
// Rows grouped by expert and brought back
// ------------------------------------------------------------------------------------------------
bool is_8_bit(at::ScalarType t) { return t == at::kFloat8_e4m3fn || t == at::kChar; }

Four moe_group_rows_cuda(const at::Tensor& x, const at::Tensor& topk_idx, int64_t num_experts, const OptTensor& scales) {
    check_operand(x, x, "x");
    check_operand(topk_idx, x, "topk_idx");
    CAM_ASSERT(x.dim() == 2 && x.size(1) >= 1 && topk_idx.dim() == 2 && topk_idx.size(0) == x.size(0), "moe_group_rows: x must be [T, h], topk_idx [T, k]");
    if (!is_8_bit(x.scalar_type())) dtype_of(x.scalar_type(), "moe_group_rows: x (where it is not float8_e4m3fn or int8)");
    CAM_ASSERT(topk_idx.scalar_type() == at::kLong || topk_idx.scalar_type() == at::kInt, "moe_group_rows: topk_idx must be int64 or int32");
    const int64_t t = x.size(0), k = topk_idx.size(1);
    CAM_ASSERT(k >= 1 && k <= 32, "moe_group_rows: ", num(k), " choices per token; 1 to 32");
    CAM_ASSERT(num_experts >= 1 && num_experts <= 1024, "moe_group_rows: ", num(num_experts), " experts; 1 to 1024");
    CAM_ASSERT(t * k < (1ll << 31) - 512 && x.size(1) < (1 << 26), "moe_group_rows: ", num(t), " tokens with ", num(k), " choices, rows of ", num(x.size(1)));
    int64_t cols = 0;
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor row_scales;
    if (given(scales)) {
        check_operand(*scales, x, "scales");
        CAM_ASSERT(scales->scalar_type() == at::kFloat && (scales->dim() == 1 || scales->dim() == 2) && scales->size(0) == t, "moe_group_rows: scales must be float32 [T] or [T, s]");
        cols = scales->dim() == 1 ? 1 : scales->size(1);
        CAM_ASSERT(cols >= 1 && cols < (1 << 26), "moe_group_rows: scales must be float32 [T] or [T, s]");
        auto of = scales->sizes().vec();
        of[0] = t * k;
        row_scales = cuda_empty(of, at::kFloat, x);
    } else {
        row_scales = cuda_empty({0}, at::kFloat, x);
    }
    at::Tensor rows = cuda_empty({t * k, x.size(1)}, x.scalar_type(), x);
    at::Tensor offsets = cuda_empty({num_experts + 1}, at::kInt, x), slots = cuda_empty({t, k}, at::kInt, x);
    CAM_RT(cam_moe_group_rows(data_or_null(x), x.size(1) * x.element_size(), static_cast<int>(x.element_size()), given(scales) ? floats_or_null(*scales) : nullptr, static_cast<int>(cols),
                              data_or_null(topk_idx), topk_idx.scalar_type() == at::kLong, t, static_cast<int>(k), static_cast<int>(num_experts),
                              data_or_null(rows), floats_or_null(row_scales), offsets.data_ptr<int>(), static_cast<int*>(data_or_null(slots)), stream_now()));
    return {rows, row_scales, offsets, slots};
}

struct UngroupProblem {
    int64_t num_rows, tokens;
    int h, k, dtype;
};

// `h` 0: the width is that of the rows
UngroupProblem check_ungroup(const char* op, const at::Tensor& rows, const at::Tensor& slots, const OptTensor& weights, int64_t h = 0) {
    check_operand(rows, rows, "rows");
    check_operand(slots, rows, "slots");
    UngroupProblem p{};
    p.dtype = dtype_of(rows.scalar_type(), "rows");
    if (h == 0 && rows.dim() == 2) h = rows.size(1);
    CAM_ASSERT(rows.dim() == 2 && h >= 1 && h < (1 << 26) && rows.size(0) < (1ll << 31) - 512, op, ": rows must be [M, h]");
    CAM_ASSERT(slots.dim() == 2 && slots.scalar_type() == at::kInt && slots.size(1) >= 1 && slots.size(1) <= 32, op, ": slots must be int32 [T, k] with k of 1 to 32");
    CAM_ASSERT(slots.numel() < (1ll << 31) - 512, op, ": ", num(slots.numel()), " slots");
    if (given(weights)) {
        check_operand(*weights, rows, "topk_weights");
        CAM_ASSERT(weights->scalar_type() == at::kFloat && weights->sizes() == slots.sizes(), op, ": topk_weights must be float32 ", shape(slots.sizes()));
    }
    p.num_rows = rows.size(0);
    p.h = static_cast<int>(h);
    p.tokens = slots.size(0);
    p.k = static_cast<int>(slots.size(1));
    return p;
}

at::Tensor moe_ungroup_rows_cuda(const at::Tensor& rows, const at::Tensor& slots, const OptTensor& weights, const OptTensor& residual) {
    const UngroupProblem p = check_ungroup("moe_ungroup_rows", rows, slots, weights);
    if (given(residual)) {
        check_operand(*residual, rows, "residual");
        CAM_ASSERT(residual->scalar_type() == rows.scalar_type() && residual->dim() == 2 && residual->size(0) == p.tokens && residual->size(1) == p.h,
                   "moe_ungroup_rows: residual must be [T, h] of the rows' type");
    }
    c10::cuda::CUDAGuard guard(rows.device());
    at::Tensor out = cuda_empty({p.tokens, p.h}, rows.scalar_type(), rows);
    if (p.tokens == 0) return out;
    CAM_RT(cam_moe_ungroup_rows(data_or_null(rows), p.dtype, p.num_rows, p.h, slots.data_ptr<int>(), p.tokens, p.k,
                                given(weights) ? weights->data_ptr<float>() : nullptr, given(residual) ? residual->data_ptr() : nullptr,
                                out.data_ptr(), stream_now()));
    return out;
}

Two moe_ungroup_rows_backward_cuda(const at::Tensor& dout, const at::Tensor& rows, const at::Tensor& slots, const OptTensor& weights,
                                   bool need_drows, bool need_dweights) {
    // gradients of rows alone need their number: rows [M, 0] will do
    const bool numbered = !need_dweights && rows.dim() == 2 && rows.size(1) == 0 && dout.dim() == 2;
    const UngroupProblem p = check_ungroup("moe_ungroup_rows_backward", rows, slots, weights, numbered ? dout.size(1) : 0);
    check_operand(dout, rows, "dout");
    CAM_ASSERT(dout.scalar_type() == rows.scalar_type() && dout.dim() == 2 && dout.size(0) == p.tokens && dout.size(1) == p.h,
               "moe_ungroup_rows_backward: dout must be [T, h] of the rows' type");
    c10::cuda::CUDAGuard guard(rows.device());
    at::Tensor drows = need_drows ? cuda_empty({p.num_rows, p.h}, rows.scalar_type(), rows) : cuda_none(rows);
    at::Tensor dw = need_dweights ? cuda_empty({p.tokens, p.k}, at::kFloat, rows) : cuda_empty({0}, at::kFloat, rows);
    const int64_t words = need_drows ? cam_moe_ungroup_rows_backward_words(p.dtype, p.num_rows, p.h, p.tokens, p.k) : 0;
    at::Tensor used = words > 0 ? cuda_empty({words}, at::kInt, rows) : at::Tensor();
    CAM_RT(cam_moe_ungroup_rows_backward(data_or_null(dout), data_or_null(rows), p.dtype, p.num_rows, p.h, static_cast<const int*>(data_or_null(slots)),
                                         p.tokens, p.k, given(weights) ? floats_or_null(*weights) : nullptr, data_or_null(drows), floats_or_null(dw),
                                         static_cast<uint32_t*>(data_or_null(used)), stream_now()));
    return {drows, dw};
}

// ------------------------------------------------------------------------------------------------
// Shapes
// ------------------------------------------------------------------------------------------------
at::Tensor rms_norm_meta(const at::Tensor& x, const at::Tensor&, double) { return at::empty_like(x); }
Two add_rms_norm_meta(const at::Tensor& x, const at::Tensor& residual, const at::Tensor&, double) { return {at::empty_like(x), at::empty_like(residual)}; }
Three rms_norm_train_meta(const at::Tensor& x, const OptTensor& residual, const at::Tensor&, double) {
    const auto n = x.sym_sizes();
    c10::SymInt rows = 1;
    for (size_t i = 0; i + 1 < n.size(); ++i) rows = rows * n[i];
    return {at::empty_like(x), given(residual) ? at::empty_like(*residual) : none_of(x), at::empty_symint({rows}, x.options().dtype(at::kFloat))};
}
Three rms_norm_backward_meta(const at::Tensor& dy, const OptTensor&, const at::Tensor& sum, const at::Tensor& weight, const at::Tensor&, bool need_dx,
                             bool need_dres, bool need_dw) {
    return norm_grads_empty([](const at::Tensor& t) { return at::empty_like(t); }, none_of, dy, sum, weight, need_dx, need_dres, need_dw);
}
Four rms_norm_quant_meta(const at::Tensor& x, const at::Tensor&, int64_t quant_mode, const OptTensor& residual, double, bool with_rows) {
    const at::ScalarType qt = norm_quant_type(quant_mode);
    auto scales_of = x.sym_sizes().vec();
    if (quant_mode == 2) scales_of.pop_back();
    else scales_of.back() = scales_of.back() / 128;
    return {at::empty_symint(x.sym_sizes(), x.options().dtype(qt)), at::empty_symint(scales_of, x.options().dtype(at::kFloat)),
            given(residual) ? at::empty_like(*residual) : none_of(x), with_rows ? at::empty_like(x) : none_of(x)};
}
Two moe_route_meta(const at::Tensor& logits, int64_t k, const OptTensor&, c10::string_view, int64_t, int64_t, int64_t, bool, double) {
    return {at::empty_symint({logits.sym_size(0), k}, logits.options().dtype(at::kLong)), at::empty_symint({logits.sym_size(0), k}, logits.options().dtype(at::kFloat))};
}
at::Tensor moe_route_backward_meta(const at::Tensor&, const at::Tensor& logits, const at::Tensor&, c10::string_view, bool, double) { return at::empty_like(logits); }
Four moe_group_rows_meta(const at::Tensor& x, const at::Tensor& topk_idx, int64_t num_experts, const OptTensor& scales) {
    const c10::SymInt pairs = topk_idx.sym_size(0) * topk_idx.sym_size(1);
    at::Tensor row_scales = at::empty({0}, x.options().dtype(at::kFloat));
    if (given(scales)) {
        auto of = scales->sym_sizes().vec();
        of[0] = pairs;
        row_scales = at::empty_symint(of, scales->options());
    }
    const auto ints = x.options().dtype(at::kInt);
    return {at::empty_symint({pairs, x.sym_size(1)}, x.options()), row_scales, at::empty({num_experts + 1}, ints), at::empty_symint(topk_idx.sym_sizes(), ints)};
}
at::Tensor moe_ungroup_rows_meta(const at::Tensor& rows, const at::Tensor& slots, const OptTensor&, const OptTensor&) {
    return at::empty_symint({slots.sym_size(0), rows.sym_size(1)}, rows.options());
}
Two moe_ungroup_rows_backward_meta(const at::Tensor& dout, const at::Tensor& rows, const at::Tensor& slots, const OptTensor&, bool need_drows, bool need_dweights) {
    const auto floats = rows.options().dtype(at::kFloat);
    return {need_drows ? at::empty_symint({rows.sym_size(0), dout.sym_size(1)}, rows.options()) : none_of(rows), need_dweights ? at::empty_symint(slots.sym_sizes(), floats) : at::empty({0}, floats)};
}

// ------------------------------------------------------------------------------------------------
// Gradients
// ------------------------------------------------------------------------------------------------
template <class Function>
auto find_op(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Function>();
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

at::Tensor or_undefined(const OptTensor& t) { return given(t) ? *t : at::Tensor(); }

struct RmsNormFunction : public torch::autograd::Function<RmsNormFunction> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& residual, const at::Tensor& weight, double eps) {
        at::AutoDispatchBelowADInplaceOrView guard;
        static auto op = find_op<Three(const at::Tensor&, const OptTensor&, const at::Tensor&, double)>("umdk_cam_op_lib::rms_norm_train");
        auto [y, sum, rstd] = op.call(x, residual, weight, eps);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({given(residual) ? sum : kept_for_backward(x), weight, rstd});
        if (given(residual)) return {y, sum};
        return {y};
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        static auto op = find_op<Three(const at::Tensor&, const OptTensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, bool, bool, bool)>(
            "umdk_cam_op_lib::rms_norm_backward");
        // needs_input_grad counts the tensors that were given
        const bool with = grads.size() > 1;
        const bool need_dx = ctx->needs_input_grad(0), need_dres = with && ctx->needs_input_grad(1), need_dw = ctx->needs_input_grad(with ? 2 : 1);
        const at::Tensor dy = grads[0], ds = with ? grads[1] : at::Tensor();
        if (!dy.defined() && !ds.defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
        const auto s = ctx->get_saved_variables();
        // the sum alone is used; autograd brings its gradient to x's type
        if (!dy.defined()) return {need_dx ? ds : at::Tensor(), need_dres ? ds : at::Tensor(), need_dw ? at::zeros_like(s[1]) : at::Tensor(), at::Tensor()};
        BackwardGuard guard;
        auto [dx, dres, dw] = op.call(dy.contiguous(), ds.defined() ? OptTensor(ds.contiguous()) : OptTensor(), s[0], s[1], s[2], need_dx, need_dres, need_dw);
        const bool one = dy.scalar_type() == s[0].scalar_type();
        return {need_dx ? dx : at::Tensor(), need_dres ? (one ? dx : dres) : at::Tensor(), need_dw ? dw : at::Tensor(), at::Tensor()};
    }
};

at::Tensor rms_norm_autograd(const at::Tensor& x, const at::Tensor& weight, double eps) {
    if (records_graph("rms_norm", {{&x, "x"}, {&weight, "weight"}})) return RmsNormFunction::apply(x, OptTensor(), weight, eps)[0];
    at::AutoDispatchBelowADInplaceOrView guard;
    static auto op = find_op<at::Tensor(const at::Tensor&, const at::Tensor&, double)>("umdk_cam_op_lib::rms_norm");
    return op.call(x, weight, eps);
}

Two add_rms_norm_autograd(const at::Tensor& x, const at::Tensor& residual, const at::Tensor& weight, double eps) {
    if (records_graph("add_rms_norm", {{&x, "x"}, {&residual, "residual"}, {&weight, "weight"}})) {
        auto out = RmsNormFunction::apply(x, OptTensor(residual), weight, eps);
        return {out[0], out[1]};
    }
    at::AutoDispatchBelowADInplaceOrView guard;
    static auto op = find_op<Two(const at::Tensor&, const at::Tensor&, const at::Tensor&, double)>("umdk_cam_op_lib::add_rms_norm");
    return op.call(x, residual, weight, eps);
}

using RouteOp = Two(const at::Tensor&, int64_t, const OptTensor&, c10::string_view, int64_t, int64_t, int64_t, bool, double);

Two call_route(const at::Tensor& logits, int64_t k, const OptTensor& bias, c10::string_view score, int64_t num_groups, int64_t topk_groups,
               int64_t group_top, bool renormalize, double scale) {
    static auto op = find_op<RouteOp>("umdk_cam_op_lib::moe_route");
    return op.call(logits, k, bias, score, num_groups, topk_groups, group_top, renormalize, scale);
}

struct RouteFunction : public torch::autograd::Function<RouteFunction> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, int64_t k, const OptTensor& bias, const std::string& score,
                                 int64_t num_groups, int64_t topk_groups, int64_t group_top, bool renormalize, double scale) {
        at::AutoDispatchBelowADInplaceOrView guard;
        auto [idx, w] = call_route(logits, k, bias, score, num_groups, topk_groups, group_top, renormalize, scale);
        ctx->set_materialize_grads(false);
        ctx->mark_non_differentiable({idx});
        ctx->save_for_backward({kept_for_backward(logits), idx});
        ctx->saved_data["plan"] = std::vector<double>{score == "sigmoid" ? 1.0 : 0.0, renormalize ? 1.0 : 0.0, scale};
        return {idx, w};
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        static auto op = find_op<at::Tensor(const at::Tensor&, const at::Tensor&, const at::Tensor&, c10::string_view, bool, double)>("umdk_cam_op_lib::moe_route_backward");
        variable_list out(9);
        if (!grads[1].defined()) return out;
        const auto s = ctx->get_saved_variables();
        const auto plan = ctx->saved_data["plan"].toDoubleVector();
        BackwardGuard guard;
        out[0] = op.call(grads[1].contiguous(), s[0], s[1], plan[0] != 0.0 ? "sigmoid" : "softmax", plan[1] != 0.0, plan[2]);
        return out;
    }
};

Two moe_route_autograd(const at::Tensor& logits, int64_t k, const OptTensor& bias, c10::string_view score, int64_t num_groups, int64_t topk_groups,
                       int64_t group_top, bool renormalize, double scale) {
    if (records_graph("moe_route", {{&logits, "logits"}})) {
        auto out = RouteFunction::apply(logits, k, given(bias) ? OptTensor(bias->detach()) : bias, std::string(score.data(), score.size()), num_groups, topk_groups,
                                        group_top, renormalize, scale);
        return {out[0], out[1]};
    }
    at::AutoDispatchBelowADInplaceOrView guard;
    return call_route(logits, k, bias, score, num_groups, topk_groups, group_top, renormalize, scale);
}

using GroupOp = Four(const at::Tensor&, const at::Tensor&, int64_t, const OptTensor&);
using UngroupOp = at::Tensor(const at::Tensor&, const at::Tensor&, const OptTensor&, const OptTensor&);

Four call_group(const at::Tensor& x, const at::Tensor& topk_idx, int64_t num_experts, const OptTensor& scales) {
    static auto op = find_op<GroupOp>("umdk_cam_op_lib::moe_group_rows");
    return op.call(x, topk_idx, num_experts, scales);
}
at::Tensor call_ungroup(const at::Tensor& rows, const at::Tensor& slots, const OptTensor& weights, const OptTensor& residual) {
    static auto op = find_op<UngroupOp>("umdk_cam_op_lib::moe_ungroup_rows");
    return op.call(rows, slots, weights, residual);
}

struct GroupRowsFunction : public torch::autograd::Function<GroupRowsFunction> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& topk_idx, int64_t num_experts, const OptTensor& scales) {
        at::AutoDispatchBelowADInplaceOrView guard;
        auto [rows, row_scales, offsets, slots] = call_group(x, topk_idx, num_experts, scales);
        ctx->set_materialize_grads(false);
        ctx->mark_non_differentiable({row_scales, offsets, slots});
        ctx->save_for_backward({slots});
        return {rows, row_scales, offsets, slots};
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        variable_list out(4);
        BackwardGuard guard;
        if (grads[0].defined()) out[0] = call_ungroup(grads[0].contiguous(), ctx->get_saved_variables()[0], OptTensor(), OptTensor());
        return out;
    }
};

Four moe_group_rows_autograd(const at::Tensor& x, const at::Tensor& topk_idx, int64_t num_experts, const OptTensor& scales) {
    if (records_graph("moe_group_rows", {{&x, "x"}})) {
        CAM_ASSERT(!is_8_bit(x.scalar_type()), "moe_group_rows: rows of 8 bits have no gradient");
        CAM_ASSERT(!given(scales) || !scales->requires_grad(), "moe_group_rows: scales have no gradient");
        auto out = GroupRowsFunction::apply(x, topk_idx, num_experts, scales);
        return {out[0], out[1], out[2], out[3]};
    }
    CAM_ASSERT(!given(scales) || !(at::GradMode::is_enabled() && scales->requires_grad()), "moe_group_rows: scales have no gradient");
    at::AutoDispatchBelowADInplaceOrView guard;
    return call_group(x, topk_idx, num_experts, scales);
}

struct UngroupRowsFunction : public torch::autograd::Function<UngroupRowsFunction> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& rows, const at::Tensor& slots, const OptTensor& weights, const OptTensor& residual) {
        at::AutoDispatchBelowADInplaceOrView guard;
        at::Tensor out = call_ungroup(rows, slots, weights, residual);
        // the rows themselves enter the gradient of the weights only; without it their number does, and they are free to change or go
        const bool rows_read = given(weights) && weights->requires_grad();
        variable_list kept = {rows_read ? kept_for_backward(rows) : at::empty_symint({rows.sym_size(0), 0}, rows.options()), kept_for_backward(slots),
                              given(weights) ? kept_for_backward(*weights) : at::Tensor()};
        if (given(residual)) kept.emplace_back();  // its place says that there was one
        ctx->save_for_backward(kept);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        static auto op = find_op<Two(const at::Tensor&, const at::Tensor&, const at::Tensor&, const OptTensor&, bool, bool)>("umdk_cam_op_lib::moe_ungroup_rows_backward");
        variable_list out(4);
        if (!grads[0].defined()) return out;
        const auto s = ctx->get_saved_variables();
        // needs_input_grad counts the tensors that were given
        const bool weighted = s[2].defined(), residual = s.size() > 3;
        const bool need_rows = ctx->needs_input_grad(0), need_weights = weighted && ctx->needs_input_grad(2);
        if (need_rows || need_weights) {
            BackwardGuard guard;
            auto [drows, dw] = op.call(grads[0].contiguous(), s[0], s[1], s[2].defined() ? OptTensor(s[2]) : OptTensor(), need_rows, need_weights);
            if (need_rows) out[0] = drows;
            if (need_weights) out[2] = dw;
        }
        if (residual && ctx->needs_input_grad(weighted ? 3 : 2)) out[3] = grads[0];
        return out;
    }
};

at::Tensor moe_ungroup_rows_autograd(const at::Tensor& rows, const at::Tensor& slots, const OptTensor& weights, const OptTensor& residual) {
    const at::Tensor w = or_undefined(weights), r = or_undefined(residual);
    if (records_graph("moe_ungroup_rows", {{&rows, "rows"}, {&w, "topk_weights"}, {&r, "residual"}})) return UngroupRowsFunction::apply(rows, slots, weights, residual);
    at::AutoDispatchBelowADInplaceOrView guard;
    return call_ungroup(rows, slots, weights, residual);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(umdk_cam_op_lib, m) {
    m.def("rms_norm(Tensor x, Tensor weight, float eps=1e-6) -> Tensor");
    m.def("add_rms_norm(Tensor x, Tensor residual, Tensor weight, float eps=1e-6) -> (Tensor, Tensor)");
    m.def("rms_norm_train(Tensor x, Tensor? residual, Tensor weight, float eps=1e-6) -> (Tensor, Tensor, Tensor)");
    m.def("rms_norm_backward(Tensor dy, Tensor? dsum, Tensor sum, Tensor weight, Tensor rstd, bool need_dx=True, bool need_dresidual=True, "
          "bool need_dweight=True) -> (Tensor, Tensor, Tensor)");
    m.def("rms_norm_quant(Tensor x, Tensor weight, int quant_mode, Tensor? residual=None, float eps=1e-6, bool with_rows=False) -> "
          "(Tensor, Tensor, Tensor, Tensor)");
    m.def("moe_route(Tensor logits, int k, Tensor? bias=None, str score=\"softmax\", int num_groups=1, int topk_groups=1, int group_top=1, "
          "bool renormalize=True, float scale=1.0) -> (Tensor, Tensor)");
    m.def("moe_route_backward(Tensor dweights, Tensor logits, Tensor topk_idx, str score=\"softmax\", bool renormalize=True, float scale=1.0) "
          "-> Tensor");
    m.def("moe_group_rows(Tensor x, Tensor topk_idx, int num_experts, Tensor? scales=None) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("moe_ungroup_rows(Tensor rows, Tensor slots, Tensor? topk_weights=None, Tensor? residual=None) -> Tensor");
    m.def("moe_ungroup_rows_backward(Tensor dout, Tensor rows, Tensor slots, Tensor? topk_weights=None, bool need_drows=True, "
          "bool need_dweights=True) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(umdk_cam_op_lib, CUDA, m) {
    m.impl("rms_norm", &rms_norm_cuda);
    m.impl("add_rms_norm", &add_rms_norm_cuda);
    m.impl("rms_norm_train", &rms_norm_train_cuda);
    m.impl("rms_norm_backward", &rms_norm_backward_cuda);
    m.impl("rms_norm_quant", &rms_norm_quant_cuda);
    m.impl("moe_route", &moe_route_cuda);
    m.impl("moe_route_backward", &moe_route_backward_cuda);
    m.impl("moe_group_rows", &moe_group_rows_cuda);
    m.impl("moe_ungroup_rows", &moe_ungroup_rows_cuda);
    m.impl("moe_ungroup_rows_backward", &moe_ungroup_rows_backward_cuda);
}

TORCH_LIBRARY_IMPL(umdk_cam_op_lib, Meta, m) {
    m.impl("rms_norm", &rms_norm_meta);
    m.impl("add_rms_norm", &add_rms_norm_meta);
    m.impl("rms_norm_train", &rms_norm_train_meta);
    m.impl("rms_norm_backward", &rms_norm_backward_meta);
    m.impl("rms_norm_quant", &rms_norm_quant_meta);
    m.impl("moe_route", &moe_route_meta);
    m.impl("moe_route_backward", &moe_route_backward_meta);
    m.impl("moe_group_rows", &moe_group_rows_meta);
    m.impl("moe_ungroup_rows", &moe_ungroup_rows_meta);
    m.impl("moe_ungroup_rows_backward", &moe_ungroup_rows_backward_meta);
}

TORCH_LIBRARY_IMPL(umdk_cam_op_lib, Autograd, m) {
    m.impl("rms_norm", &rms_norm_autograd);
    m.impl("add_rms_norm", &add_rms_norm_autograd);
    m.impl("moe_route", &moe_route_autograd);
    m.impl("moe_group_rows", &moe_group_rows_autograd);
    m.impl("moe_ungroup_rows", &moe_ungroup_rows_autograd);
    for (const char* name : {"rms_norm_train", "rms_norm_backward", "rms_norm_quant", "moe_route_backward", "moe_ungroup_rows_backward"})
        m.impl(name, torch::autograd::autogradNotImplementedFallback());
}
