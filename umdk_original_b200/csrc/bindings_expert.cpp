// PyTorch bindings of the expert-MLP operators that need no Buffer: 4-bit quantisation, grouped products of 4-bit operands, the
// gated feed-forward block of 16-bit experts with its backward pass.
// Schemas are added to the library that bindings.cpp defines.
#include "bindings_common.h"
#include "runtime/expert_ops.h"

namespace {

using namespace umdk;

at::ScalarType scale_type(int64_t block) {
    CAM_ASSERT(block == 16 || block == 32, "block must be 16 (nvfp4) or 32 (mxfp4), got ", num(block));
    return block == 16 ? at::kFloat8_e4m3fn : at::kFloat8_e8m0fnu;
}

// Block of a scale tensor, by its type.
int64_t block_of(const at::Tensor& s, const char* what) {
    CAM_ASSERT(s.scalar_type() == at::kFloat8_e4m3fn || s.scalar_type() == at::kFloat8_e8m0fnu, what,
               " must be float8_e4m3fn (nvfp4) or float8_e8m0fnu (mxfp4)");
    return s.scalar_type() == at::kFloat8_e4m3fn ? 16 : 32;
}

// Codes [..., K/2] with their scales [..., K/block]; returns K.
int64_t check_fp4(const at::Tensor& q, const at::Tensor& s, int64_t block, const char* what) {
    CAM_ASSERT(q.scalar_type() == at::kByte && q.dim() >= 1, what, " codes must be uint8 [..., K / 2]");
    const int64_t k = q.size(-1) * 2;
    CAM_ASSERT(k % block == 0, what, ": K ", num(k), " is not a multiple of the block ", num(block));
    auto want = q.sizes().vec();
    want.back() = k / block;
    CAM_ASSERT(s.sizes() == at::IntArrayRef(want), what, " scales must be [..., K / ", num(block), "] for codes [..., K / 2]: got ",
               shape(s.sizes()), " for ", shape(q.sizes()));
    return k;
}

// A global scale: one float, or (where `per` > 0) one for each of `per` experts.  Only nvfp4 has them.
const float* check_gscale(const OptTensor& g, const at::Tensor& with, int64_t block, int64_t per, const char* what) {
    if (!given(g)) return nullptr;
    CAM_ASSERT(block == 16, what, ": mxfp4 has no global scale");
    check_operand(*g, with, what);
    CAM_ASSERT(g->scalar_type() == at::kFloat && (per > 0 ? g->numel() == per : g->numel() == 1), what, " must be float32 with ",
               num(per > 0 ? per : 1), " element(s)");
    return g->data_ptr<float>();
}

std::tuple<at::Tensor, at::Tensor> quantize_fp4_empty(const at::Tensor& x, int64_t block) {
    const auto st = scale_type(block);
    CAM_ASSERT(x.dim() >= 1 && x.size(-1) % block == 0 && x.size(-1) > 0, "quantize_fp4: the last dimension must be a multiple of ", num(block));
    auto qs = x.sizes().vec(), ss = x.sizes().vec();
    qs.back() /= 2;
    ss.back() /= block;
    return {at::empty(qs, x.options().dtype(at::kByte)), at::empty(ss, x.options().dtype(st))};
}

// Global scales of a tensor: one, or one per leading index of a 3-D tensor (experts).
int64_t gscales_of(const OptTensor& g, const at::Tensor& t) { return given(g) && t.dim() == 3 && g->numel() != 1 ? t.size(0) : 0; }

std::tuple<at::Tensor, at::Tensor> quantize_fp4_cuda(const at::Tensor& x, int64_t block, const OptTensor& global_scale) {
    check_operand(x, x, "x");
    const int dt = dtype_of(x.scalar_type(), "x");
    const int64_t per = gscales_of(global_scale, x);
    const float* g = check_gscale(global_scale, x, block, per, "global_scale");
    c10::cuda::CUDAGuard guard(x.device());
    auto out = quantize_fp4_empty(x, block);
    CAM_RT(cam_quantize_fp4(x.data_ptr(), dt, block == 16 ? 0 : 1, std::get<0>(out).data_ptr(), std::get<1>(out).data_ptr(), x.numel(), g,
                            per > 0 ? per : 1, at::cuda::getCurrentCUDAStream().stream()));
    return out;
}

at::Tensor dequantize_fp4_empty(const at::Tensor& q, c10::optional<at::ScalarType> dtype) {
    auto shape = q.sizes().vec();
    shape.back() *= 2;
    return at::empty(shape, q.options().dtype(dtype.value_or(at::kBFloat16)));
}

at::Tensor dequantize_fp4_cuda(const at::Tensor& q, const at::Tensor& s, const OptTensor& global_scale, c10::optional<at::ScalarType> dtype) {
    check_operand(q, q, "q");
    check_operand(s, q, "s");
    const int64_t block = block_of(s, "s");
    check_fp4(q, s, block, "dequantize_fp4:");
    const int64_t per = gscales_of(global_scale, q);
    const float* g = check_gscale(global_scale, q, block, per, "global_scale");
    const int dt = dtype_of(dtype.value_or(at::kBFloat16), "dtype");
    c10::cuda::CUDAGuard guard(q.device());
    at::Tensor out = dequantize_fp4_empty(q, dtype);
    CAM_RT(cam_dequantize_fp4(q.data_ptr(), s.data_ptr(), dt, block == 16 ? 0 : 1, out.data_ptr(), out.numel(), g, per > 0 ? per : 1,
                              at::cuda::getCurrentCUDAStream().stream()));
    return out;
}

struct Fp4Problem {
    int64_t rows, experts, n, k, block;
    const float *a_gs, *w_gs;
};

Fp4Problem check_grouped_fp4(const at::Tensor& a_q, const at::Tensor& a_s, const at::Tensor& w_q, const at::Tensor& w_s,
                             const at::Tensor& expert_offsets, const OptTensor& a_gs, const OptTensor& w_gs, int64_t n_step) {
    check_operand(a_q, a_q, "a_q");
    check_operand(a_s, a_q, "a_s");
    check_operand(w_q, a_q, "w_q");
    check_operand(w_s, a_q, "w_s");
    check_operand(expert_offsets, a_q, "expert_offsets");
    Fp4Problem p{};
    p.block = block_of(a_s, "a_s");
    CAM_ASSERT(block_of(w_s, "w_s") == p.block, "a_s and w_s must be of the same format");
    CAM_ASSERT(a_q.dim() == 2 && w_q.dim() == 3 && a_q.size(1) == w_q.size(2), "a_q must be [M, K / 2] and w_q [E, N, K / 2]");
    p.k = check_fp4(a_q, a_s, p.block, "a");
    check_fp4(w_q, w_s, p.block, "w");
    p.rows = a_q.size(0);
    p.experts = w_q.size(0);
    p.n = w_q.size(1);
    CAM_ASSERT(p.k % 128 == 0 && p.k > 0, "K ", num(p.k), " must be a multiple of 128");
    CAM_ASSERT(p.n % n_step == 0 && p.n > 0, "N ", num(p.n), " must be a multiple of ", num(n_step));
    CAM_ASSERT(p.experts >= 1 && p.rows < (1ll << 31) && p.experts * p.n < (1ll << 31), "M, E and E * N must be below 2^31");
    CAM_ASSERT(expert_offsets.scalar_type() == at::kInt && expert_offsets.numel() == p.experts + 1, "expert_offsets must be int32 [E+1]");
    p.a_gs = check_gscale(a_gs, a_q, p.block, 0, "a_global_scale");
    p.w_gs = check_gscale(w_gs, a_q, p.block, p.experts, "w_global_scale");
    return p;
}

at::Tensor grouped_gemm_fp4_cuda(const at::Tensor& a_q, const at::Tensor& a_s, const at::Tensor& w_q, const at::Tensor& w_s,
                                 const at::Tensor& expert_offsets, const OptTensor& a_gs, const OptTensor& w_gs) {
    const Fp4Problem p = check_grouped_fp4(a_q, a_s, w_q, w_s, expert_offsets, a_gs, w_gs, 128);
    c10::cuda::CUDAGuard guard(a_q.device());
    at::Tensor out = at::empty({p.rows, p.n}, a_q.options().dtype(at::kBFloat16));
    if (p.rows == 0) return out;
    CAM_RT(cam_grouped_gemm_fp4(a_q.data_ptr(), a_s.data_ptr(), static_cast<int>(p.rows), w_q.data_ptr(), w_s.data_ptr(),
                                expert_offsets.data_ptr<int>(), static_cast<int>(p.experts), static_cast<int>(p.n), static_cast<int>(p.k),
                                p.block == 16 ? 0 : 1, 0, p.a_gs, p.w_gs, nullptr, out.data_ptr(), nullptr,
                                at::cuda::getCurrentCUDAStream().stream()));
    return out;
}

std::tuple<at::Tensor, at::Tensor> grouped_gemm_fp4_swiglu_cuda(const at::Tensor& a_q, const at::Tensor& a_s, const at::Tensor& w_q,
                                                                const at::Tensor& w_s, const at::Tensor& expert_offsets,
                                                                const OptTensor& a_gs, const OptTensor& w_gs, const OptTensor& out_gs) {
    const Fp4Problem p = check_grouped_fp4(a_q, a_s, w_q, w_s, expert_offsets, a_gs, w_gs, 256);
    const float* og = check_gscale(out_gs, a_q, p.block, 0, "out_global_scale");
    c10::cuda::CUDAGuard guard(a_q.device());
    at::Tensor q = at::empty({p.rows, p.n / 4}, a_q.options());
    at::Tensor s = at::empty({p.rows, p.n / 2 / p.block}, a_s.options());
    if (p.rows == 0) return {q, s};
    CAM_RT(cam_grouped_gemm_fp4(a_q.data_ptr(), a_s.data_ptr(), static_cast<int>(p.rows), w_q.data_ptr(), w_s.data_ptr(),
                                expert_offsets.data_ptr<int>(), static_cast<int>(p.experts), static_cast<int>(p.n), static_cast<int>(p.k),
                                p.block == 16 ? 0 : 1, 1, p.a_gs, p.w_gs, og, q.data_ptr(), s.data_ptr(),
                                at::cuda::getCurrentCUDAStream().stream()));
    return {q, s};
}

std::tuple<at::Tensor, at::Tensor> quantize_fp4_meta(const at::Tensor& x, int64_t block, const OptTensor&) { return quantize_fp4_empty(x, block); }
at::Tensor dequantize_fp4_meta(const at::Tensor& q, const at::Tensor&, const OptTensor&, c10::optional<at::ScalarType> dtype) {
    return dequantize_fp4_empty(q, dtype);
}
at::Tensor grouped_gemm_fp4_meta(const at::Tensor& a_q, const at::Tensor&, const at::Tensor& w_q, const at::Tensor&, const at::Tensor&,
                                 const OptTensor&, const OptTensor&) {
    return at::empty({a_q.size(0), w_q.size(1)}, a_q.options().dtype(at::kBFloat16));
}
std::tuple<at::Tensor, at::Tensor> grouped_gemm_fp4_swiglu_meta(const at::Tensor& a_q, const at::Tensor& a_s, const at::Tensor& w_q,
                                                                const at::Tensor&, const at::Tensor&, const OptTensor&, const OptTensor&,
                                                                const OptTensor&) {
    return {at::empty({a_q.size(0), w_q.size(1) / 4}, a_q.options()),
            at::empty({a_q.size(0), w_q.size(1) / 2 / block_of(a_s, "a_s")}, a_s.options())};
}

// ------------------------------------------------------------------------------------------------
// Gated feed-forward block of 16-bit experts
// ------------------------------------------------------------------------------------------------
struct MlpProblem {
    int rows, experts, h, inter, dtype;
};

MlpProblem check_mlp(const at::Tensor& x, const at::Tensor& w1, const at::Tensor& w2, const at::Tensor& expert_offsets) {
    check_operand(x, x, "x");
    check_operand(w1, x, "w1");
    check_operand(w2, x, "w2");
    check_operand(expert_offsets, x, "expert_offsets");
    CAM_ASSERT(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "grouped_mlp: x must be bfloat16 or float16");
    CAM_ASSERT(w1.scalar_type() == x.scalar_type() && w2.scalar_type() == x.scalar_type(), "grouped_mlp: x, w1 and w2 must be of one type");
    CAM_ASSERT(x.dim() == 2 && w1.dim() == 3 && w2.dim() == 3, "grouped_mlp: x must be [M, h], w1 [E, 2I, h], w2 [E, h, I]");
    const int64_t m = x.size(0), h = x.size(1), e = w1.size(0), i = w2.size(2);
    CAM_ASSERT(w1.size(1) == 2 * i && w1.size(2) == h && w2.size(0) == e && w2.size(1) == h,
               "grouped_mlp: x must be [M, h], w1 [E, 2I, h], w2 [E, h, I]: got ", shape(x.sizes()), ", ", shape(w1.sizes()), ", ", shape(w2.sizes()));
    CAM_ASSERT(h > 0 && i > 0 && h % 8 == 0 && i % 8 == 0, "grouped_mlp: h ", num(h), " and I ", num(i), " must be multiples of 8");
    CAM_ASSERT(e >= 1 && m < (1ll << 31) - 512 && h < (1 << 28) && i < (1 << 28) && e < (1 << 24), "grouped_mlp: sizes out of range");
    CAM_ASSERT(expert_offsets.scalar_type() == at::kInt && expert_offsets.numel() == e + 1, "expert_offsets must be int32 [E+1]");
    return {static_cast<int>(m), static_cast<int>(e), static_cast<int>(h), static_cast<int>(i), x.scalar_type() == at::kHalf ? 1 : 0};
}

// gate_up is kept (fp32 [M, 2I]) for a backward pass, otherwise empty
std::tuple<at::Tensor, at::Tensor, at::Tensor> mlp_forward(const at::Tensor& x, const at::Tensor& w1, const at::Tensor& w2,
                                                           const at::Tensor& expert_offsets, bool keep) {
    const MlpProblem p = check_mlp(x, w1, w2, expert_offsets);
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor act = at::empty({p.rows, p.inter}, x.options());
    at::Tensor gu = at::empty({keep ? p.rows : 0, 2 * p.inter}, x.options().dtype(at::kFloat));
    at::Tensor y = at::empty({p.rows, p.h}, x.options());
    if (p.rows == 0) return {y, act, gu};
    const auto stream = at::cuda::getCurrentCUDAStream().stream();
    const int* off = expert_offsets.data_ptr<int>();
    CAM_RT(cam_grouped_mlp_up(x.data_ptr(), w1.data_ptr(), off, p.rows, p.experts, p.h, p.inter, p.dtype, act.data_ptr(),
                              keep ? gu.data_ptr<float>() : nullptr, stream));
    CAM_RT(cam_grouped_mlp_down(act.data_ptr(), w2.data_ptr(), off, p.rows, p.experts, p.h, p.inter, p.dtype, y.data_ptr(), stream));
    return {y, act, gu};
}

at::Tensor grouped_mlp_cuda(const at::Tensor& x, const at::Tensor& w1, const at::Tensor& w2, const at::Tensor& expert_offsets) {
    return std::get<0>(mlp_forward(x, w1, w2, expert_offsets, false));
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> grouped_mlp_train_cuda(const at::Tensor& x, const at::Tensor& w1, const at::Tensor& w2,
                                                                      const at::Tensor& expert_offsets) {
    return mlp_forward(x, w1, w2, expert_offsets, true);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> mlp_grads_empty(const at::Tensor& x, const at::Tensor& w1, const at::Tensor& w2,
                                                               bool need_dx, bool need_dw1, bool need_dw2) {
    auto like = [](const at::Tensor& t, bool need) { return need ? at::empty_like(t) : at::empty({0}, t.options()); };
    return {like(x, need_dx), like(w1, need_dw1), like(w2, need_dw2)};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> grouped_mlp_backward_cuda(const at::Tensor& dy_in, const at::Tensor& x, const at::Tensor& w1,
                                                                         const at::Tensor& w2, const at::Tensor& expert_offsets,
                                                                         const at::Tensor& act, const at::Tensor& gate_up, bool need_dx,
                                                                         bool need_dw1, bool need_dw2) {
    const MlpProblem p = check_mlp(x, w1, w2, expert_offsets);
    check_operand(dy_in, x, "dy");
    c10::cuda::CUDAGuard guard(x.device());
    // autograd hands out slices of larger gradients, at any offset: the caller has no say in it
    const at::Tensor dy = reinterpret_cast<uintptr_t>(dy_in.data_ptr()) % 16 == 0 ? dy_in : dy_in.clone();
    check_operand(act, x, "act");
    check_operand(gate_up, x, "gate_up");
    CAM_ASSERT(dy.scalar_type() == x.scalar_type() && dy.sizes() == x.sizes(), "grouped_mlp: dy must be like x");
    CAM_ASSERT(act.scalar_type() == x.scalar_type() && act.dim() == 2 && act.size(0) == p.rows && act.size(1) == p.inter, "grouped_mlp: act must be [M, I]");
    CAM_ASSERT(gate_up.scalar_type() == at::kFloat && gate_up.dim() == 2 && gate_up.size(0) == p.rows && gate_up.size(1) == 2 * p.inter,
               "grouped_mlp: gate_up must be float32 [M, 2I]");
    auto out = mlp_grads_empty(x, w1, w2, need_dx, need_dw1, need_dw2);
    auto& [dx, dw1, dw2] = out;
    if (p.rows == 0) {
        dw1.zero_();
        dw2.zero_();
        return out;
    }
    const auto stream = at::cuda::getCurrentCUDAStream().stream();
    const int* off = expert_offsets.data_ptr<int>();
    if (need_dw2)
        CAM_RT(cam_grouped_mlp_dw(dy.data_ptr(), act.data_ptr(), off, p.rows, p.experts, p.h, p.inter, p.dtype, dw2.data_ptr(), stream));
    if (!need_dx && !need_dw1) return out;
    at::Tensor dgu = at::empty({p.rows, 2 * p.inter}, x.options());
    CAM_RT(cam_grouped_mlp_dact(dy.data_ptr(), w2.data_ptr(), gate_up.data_ptr<float>(), off, p.rows, p.experts, p.h, p.inter, p.dtype,
                                dgu.data_ptr(), stream));
    if (need_dx)
        CAM_RT(cam_grouped_mlp_dx(dgu.data_ptr(), w1.data_ptr(), off, p.rows, p.experts, p.h, p.inter, p.dtype, dx.data_ptr(), stream));
    if (need_dw1)
        CAM_RT(cam_grouped_mlp_dw(dgu.data_ptr(), x.data_ptr(), off, p.rows, p.experts, 2 * p.inter, p.h, p.dtype, dw1.data_ptr(), stream));
    return out;
}

at::Tensor grouped_mlp_meta(const at::Tensor& x, const at::Tensor&, const at::Tensor&, const at::Tensor&) { return at::empty_like(x); }
std::tuple<at::Tensor, at::Tensor, at::Tensor> grouped_mlp_train_meta(const at::Tensor& x, const at::Tensor&, const at::Tensor& w2, const at::Tensor&) {
    return {at::empty_like(x), at::empty({x.size(0), w2.size(2)}, x.options()), at::empty({x.size(0), 2 * w2.size(2)}, x.options().dtype(at::kFloat))};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> grouped_mlp_backward_meta(const at::Tensor&, const at::Tensor& x, const at::Tensor& w1,
                                                                         const at::Tensor& w2, const at::Tensor&, const at::Tensor&,
                                                                         const at::Tensor&, bool need_dx, bool need_dw1, bool need_dw2) {
    return mlp_grads_empty(x, w1, w2, need_dx, need_dw1, need_dw2);
}

using Mlp3 = std::tuple<at::Tensor, at::Tensor, at::Tensor>;

Mlp3 call_mlp_train(const at::Tensor& x, const at::Tensor& w1, const at::Tensor& w2, const at::Tensor& off) {
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("umdk_cam_op_lib::grouped_mlp_train", "")
                         .typed<Mlp3(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&)>();
    return op.call(x, w1, w2, off);
}

at::Tensor grouped_mlp_keep(const at::Tensor& t) { return t.clone(); }

struct GroupedMlpFunction : public torch::autograd::Function<GroupedMlpFunction> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w1, const at::Tensor& w2,
                              const at::Tensor& expert_offsets) {
        at::AutoDispatchBelowADInplaceOrView guard;
        auto [y, act, gu] = call_mlp_train(x, w1, w2, expert_offsets);
        // x itself enters the gradient of w1 only
        ctx->save_for_backward({w1.requires_grad() ? kept_for_backward(x) : x, w1, w2, kept_for_backward(expert_offsets), act, gu});
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads) {
        static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("umdk_cam_op_lib::grouped_mlp_backward", "")
                             .typed<Mlp3(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                         const at::Tensor&, const at::Tensor&, bool, bool, bool)>();
        const bool need_dx = ctx->needs_input_grad(0), need_dw1 = ctx->needs_input_grad(1), need_dw2 = ctx->needs_input_grad(2);
        if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
        const auto s = ctx->get_saved_variables();
        auto [dx, dw1, dw2] = op.call(grads[0].contiguous(), s[0], s[1], s[2], s[3], s[4], s[5], need_dx, need_dw1, need_dw2);
        return {need_dx ? dx : at::Tensor(), need_dw1 ? dw1 : at::Tensor(), need_dw2 ? dw2 : at::Tensor(), at::Tensor()};
    }
};

at::Tensor grouped_mlp_autograd(const at::Tensor& x, const at::Tensor& w1, const at::Tensor& w2, const at::Tensor& expert_offsets) {
    if (records_graph("grouped_mlp", {{&x, "x"}, {&w1, "w1"}, {&w2, "w2"}})) return GroupedMlpFunction::apply(x, w1, w2, expert_offsets);
    at::AutoDispatchBelowADInplaceOrView guard;
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("umdk_cam_op_lib::grouped_mlp", "")
                         .typed<at::Tensor(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&)>();
    return op.call(x, w1, w2, expert_offsets);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(umdk_cam_op_lib, m) {
    m.def("quantize_fp4(Tensor x, int block=16, Tensor? global_scale=None) -> (Tensor, Tensor)");
    m.def("dequantize_fp4(Tensor q, Tensor s, Tensor? global_scale=None, ScalarType? dtype=None) -> Tensor");
    m.def("grouped_gemm_fp4(Tensor a_q, Tensor a_s, Tensor w_q, Tensor w_s, Tensor expert_offsets, "
          "Tensor? a_global_scale=None, Tensor? w_global_scale=None) -> Tensor");
    m.def("grouped_gemm_fp4_swiglu(Tensor a_q, Tensor a_s, Tensor w_q, Tensor w_s, Tensor expert_offsets, "
          "Tensor? a_global_scale=None, Tensor? w_global_scale=None, Tensor? out_global_scale=None) -> (Tensor, Tensor)");
    m.def("grouped_mlp(Tensor x, Tensor w1, Tensor w2, Tensor expert_offsets) -> Tensor");
    m.def("grouped_mlp_train(Tensor x, Tensor w1, Tensor w2, Tensor expert_offsets) -> (Tensor, Tensor, Tensor)");
    m.def("grouped_mlp_backward(Tensor dy, Tensor x, Tensor w1, Tensor w2, Tensor expert_offsets, Tensor act, Tensor gate_up, "
          "bool need_dx=True, bool need_dw1=True, bool need_dw2=True) -> (Tensor, Tensor, Tensor)");
    m.def("grouped_mlp_keep(Tensor t) -> Tensor");
}

TORCH_LIBRARY_IMPL(umdk_cam_op_lib, CompositeExplicitAutograd, m) { m.impl("grouped_mlp_keep", &grouped_mlp_keep); }

TORCH_LIBRARY_IMPL(umdk_cam_op_lib, CUDA, m) {
    m.impl("quantize_fp4", &quantize_fp4_cuda);
    m.impl("dequantize_fp4", &dequantize_fp4_cuda);
    m.impl("grouped_gemm_fp4", &grouped_gemm_fp4_cuda);
    m.impl("grouped_gemm_fp4_swiglu", &grouped_gemm_fp4_swiglu_cuda);
    m.impl("grouped_mlp", &grouped_mlp_cuda);
    m.impl("grouped_mlp_train", &grouped_mlp_train_cuda);
    m.impl("grouped_mlp_backward", &grouped_mlp_backward_cuda);
}

TORCH_LIBRARY_IMPL(umdk_cam_op_lib, Meta, m) {
    m.impl("quantize_fp4", &quantize_fp4_meta);
    m.impl("dequantize_fp4", &dequantize_fp4_meta);
    m.impl("grouped_gemm_fp4", &grouped_gemm_fp4_meta);
    m.impl("grouped_gemm_fp4_swiglu", &grouped_gemm_fp4_swiglu_meta);
    m.impl("grouped_mlp", &grouped_mlp_meta);
    m.impl("grouped_mlp_train", &grouped_mlp_train_meta);
    m.impl("grouped_mlp_backward", &grouped_mlp_backward_meta);
}

TORCH_LIBRARY_IMPL(umdk_cam_op_lib, Autograd, m) {
    m.impl("quantize_fp4", torch::autograd::autogradNotImplementedFallback());
    m.impl("dequantize_fp4", torch::autograd::autogradNotImplementedFallback());
    m.impl("grouped_gemm_fp4", torch::autograd::autogradNotImplementedFallback());
    m.impl("grouped_gemm_fp4_swiglu", torch::autograd::autogradNotImplementedFallback());
    m.impl("grouped_mlp", &grouped_mlp_autograd);
    m.impl("grouped_mlp_train", torch::autograd::autogradNotImplementedFallback());
    m.impl("grouped_mlp_backward", torch::autograd::autogradNotImplementedFallback());
    m.impl("grouped_mlp_keep", torch::autograd::autogradNotImplementedFallback());
}
