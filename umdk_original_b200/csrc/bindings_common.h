// What the bindings of the operators that need no Buffer share: checks of operands, messages, what an autograd function keeps, and
// the calls that autograd could not carry out.
#pragma once
#include <ATen/TensorSubclassLikeUtils.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>
#include <torch/library.h>

#include <initializer_list>
#include <string>
#include <tuple>
#include <utility>

#include "runtime/cam_runtime.h"

#define CAM_ASSERT(cond, ...) TORCH_CHECK(cond, "umdk_cam_op_lib: ", __VA_ARGS__)
#define CAM_RT(call) TORCH_CHECK((call) == 0, "umdk_cam_op_lib: ", cam_last_error())

namespace umdk {

using OptTensor = c10::optional<at::Tensor>;

// Numbers enter messages as text: formatting them through the string streams of TORCH_CHECK crashes in a process whose C++
// runtime libraries disagree about the locale.
inline std::string num(int64_t v) { return std::to_string(v); }
inline std::string shape(at::IntArrayRef v) {
    std::string s = "[";
    for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + num(v[i]);
    return s + "]";
}

inline bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

inline void check_operand(const at::Tensor& t, const at::Tensor& with, const char* what) {
    CAM_ASSERT(t.device() == with.device(), what, " must be on ", with.device().str(), ", the device of the rows");
    CAM_ASSERT(t.is_contiguous(), what, " must be contiguous");
}

inline int dtype_of(at::ScalarType t, const char* what) {
    CAM_ASSERT(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat, what, " must be bfloat16, float16 or float32");
    return t == at::kBFloat16 ? 0 : t == at::kHalf ? 1 : 2;
}

// What the backward pass will read of an input.  The rows of a dispatch are views of memory that the next dispatch on that Buffer
// overwrites, behind the back of autograd's version counters, and a program of several layers dispatches again before it runs
// backward: such memory (any that PyTorch's allocators do not own) is copied.  A tracer's stand-ins (torch.compile) do not know whose
// memory the traced program will see, so a traced program always copies, by an operator of this library: a plain clone may be
// removed by the compiler's passes, or moved into the backward pass, where it would come too late.
inline at::Tensor kept_for_backward(const at::Tensor& t) {
    if (at::isTensorSubclassLike(t)) {
        static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("umdk_cam_op_lib::grouped_mlp_keep", "")
                             .typed<at::Tensor(const at::Tensor&)>();
        return op.call(t);
    }
    return t.storage().unsafeGetStorageImpl()->resizable() ? t : t.clone();
}

// A captured backward pass that accumulates into a leaf whose accumulation node belongs to an eager graph (another stream) makes
// the autograd engine synchronise a stream that is not captured, which ends the process.  Refused while it can still be.
inline void check_capture(const at::Tensor& t, const char* op, const char* what) {
    if (!t.requires_grad() || !t.is_leaf() || !t.is_cuda()) return;
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(t);
    if (accumulator == nullptr) return;
    const auto stream = accumulator->stream();
    CAM_ASSERT(!stream.has_value() || *stream == at::cuda::getCurrentCUDAStream(t.device().index()).unwrap(), op, " is captured into a CUDA graph while a graph of derivatives that was recorded outside the capture still holds ",
               what, "; let go of its outputs before the capture");
}

// Whether a call of a differentiable operator records a graph; refuses tangents and captures that autograd could not carry out.
inline bool records_graph(const char* op, std::initializer_list<std::pair<const at::Tensor*, const char*>> operands) {
    bool wanted = false;
    for (const auto& [t, what] : operands) {
        if (t == nullptr || !t->defined()) continue;
        // a dual tensor need not require a gradient: without this its tangent would be dropped
        TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(/*level=*/0).defined(), "umdk_cam_op_lib: ", op, " has no forward-mode derivative");
        wanted = wanted || t->requires_grad();
    }
    if (!at::GradMode::is_enabled() || !wanted) return false;
    const at::Tensor& first = *operands.begin()->first;  // the operands of a call share a device
    if (first.is_cuda()) {
        c10::cuda::CUDAGuard guard(first.device());
        if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) {
            for (const auto& [t, what] : operands) {
                if (t != nullptr && t->defined()) check_capture(*t, op, what);
            }
        }
    }
    return true;
}

// Inside a backward pass: its own operators are called below autograd, whose fallback for operators without a derivative costs more than
// they do.  With create_graph the fallback stays in the way, and whoever differentiates again is told that there is no derivative.
struct BackwardGuard {
    c10::optional<at::AutoDispatchBelowADInplaceOrView> below;
    BackwardGuard() {
        if (!at::GradMode::is_enabled()) below.emplace();
    }
};

// Results of the CUDA implementations, which know where and what they are
inline at::Tensor cuda_empty(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& on) { return at::detail::empty_cuda(sizes, type, on.device(), c10::nullopt); }

}  // namespace umdk
