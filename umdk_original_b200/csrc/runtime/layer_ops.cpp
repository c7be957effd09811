// Host side of the operators round the experts: checks and launches.
#include "layer_ops.h"

#include <cstdarg>
#include <cstdio>

#include "../kernels/layer_ops.h"

namespace {

int refuse(const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return cam_fail(buf);
}

#define LAYER_CHECK(cond, ...)                   \
    do {                                         \
        if (!(cond)) return refuse(__VA_ARGS__); \
    } while (0)

bool type_ok(int t) { return t >= cam::kDtBf16 && t <= cam::kDtFp32; }

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int launched(int rc, const char* what) {
    return rc == 0 ? 0 : refuse("%s: launch failed: %s", what, cudaGetErrorString(static_cast<cudaError_t>(rc)));
}

constexpr int64_t kMaxRows = (1ll << 31) - 512;

}  // namespace

extern "C" int cam_rms_norm(const void* x, int dtype, const void* residual, int res_type, const void* weight, int weight_type, int64_t rows,
                            int h, float eps, void* y, void* sum, float* rstd, int quant_mode, void* q, float* scales, cudaStream_t stream) {
    LAYER_CHECK(x && weight && (residual == nullptr) == (sum == nullptr), "rms_norm: null operand");
    LAYER_CHECK(type_ok(dtype) && (weight_type == dtype || weight_type == cam::kDtFp32), "rms_norm: weight must be of x's type or float32");
    LAYER_CHECK(residual == nullptr || res_type == dtype || res_type == cam::kDtFp32, "rms_norm: residual must be of x's type or float32");
    LAYER_CHECK(rows >= 1 && rows < kMaxRows, "rms_norm: %lld rows", static_cast<long long>(rows));
    LAYER_CHECK(h >= 1 && h <= cam::kNormMaxHidden, "rms_norm: rows of %d values; 1 to %d", h, cam::kNormMaxHidden);
    LAYER_CHECK(eps >= 0.f, "rms_norm: eps must not be negative");
    LAYER_CHECK(quant_mode == 0 || (quant_mode >= 2 && quant_mode <= 4), "rms_norm: quant mode %d; 2 (int8), 3 or 4 (e4m3)", quant_mode);
    LAYER_CHECK(quant_mode != 0 ? q && scales : y != nullptr, "rms_norm: null output");
    if (quant_mode >= 3) {
        LAYER_CHECK(h % 128 == 0, "rms_norm_quant: e4m3 rows must be a multiple of 128 values, not %d", h);
        LAYER_CHECK(aligned(x) && aligned(residual) && aligned(weight) && aligned(y) && aligned(sum) && aligned(q), "rms_norm_quant: e4m3 rows need 16-byte aligned operands");
    }
    cam::RmsNormParams p{};
    p.x = x;
    p.residual = residual;
    p.weight = weight;
    p.res_type = res_type;
    p.weight_type = weight_type;
    p.rows = rows;
    p.h = h;
    p.eps = eps;
    p.y = y;
    p.sum = sum;
    p.rstd = rstd;
    p.quant_mode = quant_mode;
    p.q = q;
    p.scales = scales;
    return launched(cam_launch_rms_norm(&p, dtype, stream), "rms_norm");
}

extern "C" int cam_rms_norm_backward_parts(int64_t rows, int h) { return cam_rms_norm_backward_blocks(rows, h); }

extern "C" int cam_rms_norm_backward(const void* dy, int dtype, const void* dsum, const void* sum, int sum_type, const void* weight,
                                     int weight_type, const float* rstd, int64_t rows, int h, void* dx, void* dres, void* dweight,
                                     float* partial, int parts, cudaStream_t stream) {
    LAYER_CHECK(dy && sum && weight && rstd, "rms_norm_backward: null operand");
    LAYER_CHECK(type_ok(dtype) && (weight_type == dtype || weight_type == cam::kDtFp32) && (sum_type == dtype || sum_type == cam::kDtFp32),
                "rms_norm_backward: sum and weight must be of dy's type or float32");
    LAYER_CHECK(rows >= 1 && rows < kMaxRows && h >= 1 && h <= cam::kNormMaxHidden, "rms_norm_backward: %lld rows of %d values", static_cast<long long>(rows), h);
    LAYER_CHECK(dweight == nullptr || partial != nullptr, "rms_norm_backward: no workspace");
    LAYER_CHECK(parts >= 1 && parts <= cam_rms_norm_backward_blocks(rows, h), "rms_norm_backward: %d parts", parts);
    cam::RmsNormBackwardParams p{};
    p.dy = dy;
    p.dsum = dsum;
    p.sum = sum;
    p.weight = weight;
    p.rstd = rstd;
    p.sum_type = sum_type;
    p.weight_type = weight_type;
    p.rows = rows;
    p.h = h;
    p.dx = dx;
    p.dres = dres;
    p.dweight = dweight;
    p.partial = dweight != nullptr ? partial : nullptr;
    p.parts = parts;
    return launched(cam_launch_rms_norm_backward(&p, dtype, stream), "rms_norm_backward");
}

namespace {

int check_route(const char* what, int dtype, int64_t rows, int experts, int k) {
    LAYER_CHECK(type_ok(dtype), "%s: type %d", what, dtype);
    LAYER_CHECK(rows >= 1 && rows < kMaxRows, "%s: %lld rows", what, static_cast<long long>(rows));
    LAYER_CHECK(experts >= 1 && experts <= cam::kRouteMaxExperts, "%s: %d experts; 1 to %d", what, experts, cam::kRouteMaxExperts);
    LAYER_CHECK(k >= 1 && k <= experts && k <= cam::kLayerMaxTopk, "%s: k %d outside [1, min(%d experts, %d)]", what, k, experts, cam::kLayerMaxTopk);
    return 0;
}

}  // namespace

extern "C" int cam_moe_route(const void* logits, int dtype, int64_t rows, int experts, int k, const float* bias, int sigmoid, int groups,
                             int topk_groups, int group_top, int renormalize, float scale, int64_t* idx, float* weights, cudaStream_t stream) {
    LAYER_CHECK(logits && idx && weights, "moe_route: null operand");
    if (check_route("moe_route", dtype, rows, experts, k) != 0) return -1;
    LAYER_CHECK(groups >= 1 && groups <= 32 && experts % groups == 0, "moe_route: %d experts in %d groups; at most 32 groups of equal size", experts, groups);
    LAYER_CHECK(topk_groups >= 1 && topk_groups <= groups, "moe_route: topk_groups %d outside [1, %d]", topk_groups, groups);
    LAYER_CHECK(k <= experts / groups * topk_groups, "moe_route: k %d of the %d experts in %d groups", k, experts / groups * topk_groups, topk_groups);
    LAYER_CHECK(group_top == 1 || group_top == 2, "moe_route: group_top must be 1 or 2, got %d", group_top);
    cam::RouteParams p{};
    p.logits = logits;
    p.bias = bias;
    p.rows = rows;
    p.experts = experts;
    p.k = k;
    p.groups = groups;
    p.topk_groups = topk_groups;
    p.group_top = group_top;
    p.sigmoid = sigmoid;
    p.renormalize = renormalize;
    p.scale = scale;
    p.idx = idx;
    p.weights = weights;
    return launched(cam_launch_moe_route(&p, dtype, stream), "moe_route");
}

extern "C" int cam_moe_route_backward(const float* dweights, const void* logits, int dtype, const int64_t* idx, int64_t rows, int experts,
                                      int k, int sigmoid, int renormalize, float scale, void* dlogits, cudaStream_t stream) {
    LAYER_CHECK(dweights && logits && idx && dlogits, "moe_route_backward: null operand");
    if (check_route("moe_route_backward", dtype, rows, experts, k) != 0) return -1;
    cam::RouteParams p{};
    p.logits = logits;
    p.rows = rows;
    p.experts = experts;
    p.k = k;
    p.sigmoid = sigmoid;
    p.renormalize = renormalize;
    p.scale = scale;
    p.idx = const_cast<int64_t*>(idx);
    p.dweights = dweights;
    p.dlogits = dlogits;
    return launched(cam_launch_moe_route(&p, dtype, stream), "moe_route_backward");
}

namespace {

int check_pairs(const char* what, int64_t tokens, int k) {
    LAYER_CHECK(k >= 1 && k <= cam::kLayerMaxTopk, "%s: %d choices per token; 1 to %d", what, k, cam::kLayerMaxTopk);
    LAYER_CHECK(tokens >= 0 && tokens * k < kMaxRows, "%s: %lld tokens with %d choices", what, static_cast<long long>(tokens), k);
    return 0;
}

}  // namespace

extern "C" int cam_moe_group_rows(const void* x, int64_t row_bytes, int elem_bytes, const float* scales, int scale_cols, const void* idx, int idx_i64,
                                  int64_t tokens, int k, int experts, void* rows, float* row_scales, int* offsets, int* slots,
                                  cudaStream_t stream) {
    if (check_pairs("moe_group_rows", tokens, k) != 0) return -1;
    LAYER_CHECK(offsets != nullptr && (tokens == 0 || (x && idx && rows && slots)), "moe_group_rows: null operand");
    LAYER_CHECK(experts >= 1 && experts <= cam::kRouteMaxExperts, "moe_group_rows: %d experts; 1 to %d", experts, cam::kRouteMaxExperts);
    LAYER_CHECK(row_bytes >= 1 && row_bytes < (1ll << 28) && scale_cols >= 0 && scale_cols < (1 << 28), "moe_group_rows: rows of %lld bytes", static_cast<long long>(row_bytes));
    LAYER_CHECK(elem_bytes == 1 || elem_bytes == 2 || elem_bytes == 4, "moe_group_rows: elements of %d bytes", elem_bytes);
    LAYER_CHECK(row_bytes % elem_bytes == 0 && reinterpret_cast<uintptr_t>(x) % elem_bytes == 0 && (reinterpret_cast<uintptr_t>(rows) & 15u) == 0, "moe_group_rows: rows must be 16-byte aligned");
    LAYER_CHECK(scale_cols == 0 || tokens == 0 || (scales && row_scales), "moe_group_rows: null scales");
    cam::GroupRowsParams p{};
    p.x = x;
    p.scales = scales;
    p.idx = idx;
    p.idx_i64 = idx_i64;
    p.tokens = tokens;
    p.k = k;
    p.experts = experts;
    p.scale_cols = scale_cols;
    p.row_bytes = row_bytes;
    p.elem_bytes = elem_bytes;
    p.rows = rows;
    p.row_scales = row_scales;
    p.offsets = offsets;
    p.slots = slots;
    return launched(cam_launch_group_rows(&p, stream), "moe_group_rows");
}

namespace {

int check_ungroup(const char* what, int dtype, int64_t num_rows, int h, int64_t tokens, int k) {
    if (check_pairs(what, tokens, k) != 0) return -1;
    LAYER_CHECK(type_ok(dtype), "%s: type %d", what, dtype);
    LAYER_CHECK(num_rows >= 0 && num_rows < kMaxRows && h >= 1 && h < (1 << 28), "%s: %lld rows of %d values", what, static_cast<long long>(num_rows), h);
    return 0;
}

}  // namespace

extern "C" int cam_moe_ungroup_rows(const void* rows, int dtype, int64_t num_rows, int h, const int* slots, int64_t tokens, int k,
                                    const float* weights, const void* residual, void* out, cudaStream_t stream) {
    if (check_ungroup("moe_ungroup_rows", dtype, num_rows, h, tokens, k) != 0) return -1;
    if (tokens == 0) return 0;
    LAYER_CHECK((rows || num_rows == 0) && slots && out, "moe_ungroup_rows: null operand");
    cam::UngroupRowsParams p{};
    p.rows = rows;
    p.num_rows = num_rows;
    p.h = h;
    p.slots = slots;
    p.tokens = tokens;
    p.k = k;
    p.weights = weights;
    p.residual = residual;
    p.out = out;
    return launched(cam_launch_ungroup_rows(&p, dtype, stream), "moe_ungroup_rows");
}

extern "C" int64_t cam_moe_ungroup_rows_backward_words(int dtype, int64_t num_rows, int h, int64_t tokens, int k) {
    return cam_ungroup_rows_backward_map_words(num_rows, h, dtype, tokens * k);
}

extern "C" int cam_moe_ungroup_rows_backward(const void* dout, const void* rows, int dtype, int64_t num_rows, int h, const int* slots,
                                             int64_t tokens, int k, const float* weights, void* drows, float* dweights,
                                             uint32_t* used, cudaStream_t stream) {
    if (check_ungroup("moe_ungroup_rows_backward", dtype, num_rows, h, tokens, k) != 0) return -1;
    LAYER_CHECK(tokens == 0 || (dout && slots), "moe_ungroup_rows_backward: null operand");
    LAYER_CHECK(dweights == nullptr || rows != nullptr || num_rows == 0, "moe_ungroup_rows_backward: null rows");
    if (drows == nullptr && dweights == nullptr) return 0;
    LAYER_CHECK(drows == nullptr || used != nullptr || cam_moe_ungroup_rows_backward_words(dtype, num_rows, h, tokens, k) == 0, "moe_ungroup_rows_backward: no workspace");
    cam::UngroupRowsParams p{};
    p.rows = rows;
    p.num_rows = num_rows;
    p.h = h;
    p.slots = slots;
    p.tokens = tokens;
    p.k = k;
    p.weights = weights;
    p.dout = dout;
    p.drows = drows;
    p.dweights = dweights;
    p.used = used;
    return launched(cam_launch_ungroup_rows_backward(&p, dtype, stream), "moe_ungroup_rows_backward");
}
