// Host side of the expert-MLP operators that need no Buffer: checks, tensor maps, launches.
#include "expert_ops.h"

#include <cstdarg>
#include <cstdio>

#include "../kernels/expert_ops.h"

namespace {

int refuse(const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return cam_fail(buf);
}

#define EXP_CHECK(cond, ...)                     \
    do {                                         \
        if (!(cond)) return refuse(__VA_ARGS__); \
    } while (0)

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// [rows, bytes] with boxes of 128 bytes x box_rows
int map_2d(CUtensorMap* out, const void* base, uint64_t bytes, uint64_t rows, uint32_t box_rows) {
    const uint64_t dims[2] = {bytes, rows}, strides[1] = {bytes};
    const uint32_t box[2] = {128, box_rows};
    return cam_encode_tmap(out, base, 2, dims, strides, box);
}

int launched(int rc, const char* what) {
    return rc == 0 ? 0 : refuse("%s: launch failed: %s", what, cudaGetErrorString(static_cast<cudaError_t>(rc)));
}

}  // namespace

extern "C" int cam_quantize_fp4(const void* x, int dtype, int fmt, void* q, void* s, int64_t numel, const float* gscale,
                                int64_t gscales, cudaStream_t stream) {
    if (numel == 0) return 0;
    EXP_CHECK(x && q && s, "quantize_fp4: null operand");
    EXP_CHECK(numel > 0 && numel % (fmt == 0 ? 16 : 32) == 0, "quantize_fp4: %lld values are not whole blocks", static_cast<long long>(numel));
    EXP_CHECK(aligned(x, 16) && aligned(q, 8), "quantize_fp4: operands must be 16-byte aligned");
    const int64_t groups = numel / 16;
    EXP_CHECK(gscale == nullptr || (gscales >= 1 && groups % gscales == 0), "quantize_fp4: %lld global scales", static_cast<long long>(gscales));
    return launched(cam_launch_quantize_fp4(x, dtype, fmt, q, s, groups, gscale, gscale && gscales > 1 ? groups / gscales : 0, stream), "quantize_fp4");
}

extern "C" int cam_dequantize_fp4(const void* q, const void* s, int dtype, int fmt, void* out, int64_t numel, const float* gscale,
                                  int64_t gscales, cudaStream_t stream) {
    if (numel == 0) return 0;
    EXP_CHECK(q && s && out, "dequantize_fp4: null operand");
    EXP_CHECK(numel > 0 && numel % (fmt == 0 ? 16 : 32) == 0, "dequantize_fp4: %lld values are not whole blocks", static_cast<long long>(numel));
    EXP_CHECK(aligned(q, 8) && aligned(out, 16), "dequantize_fp4: operands must be 8-byte aligned");
    const int64_t groups = numel / 16;
    EXP_CHECK(gscale == nullptr || (gscales >= 1 && groups % gscales == 0), "dequantize_fp4: %lld global scales", static_cast<long long>(gscales));
    return launched(cam_launch_dequantize_fp4(q, s, dtype, fmt, out, groups, gscale, gscale && gscales > 1 ? groups / gscales : 0, stream), "dequantize_fp4");
}

extern "C" int cam_grouped_gemm_fp4(const void* a_q, const void* a_s, int rows, const void* w_q, const void* w_s, const int* offsets,
                                    int num_experts, int n_dim, int k_dim, int fmt, int swiglu, const float* a_gscale,
                                    const float* w_gscale, const float* out_gscale, void* out, void* out_s, cudaStream_t stream) {
    EXP_CHECK(a_q && a_s && w_q && w_s && offsets && out && (!swiglu || out_s), "grouped_gemm_fp4: null operand");
    EXP_CHECK(rows >= 1 && num_experts >= 1, "grouped_gemm_fp4: empty problem");
    EXP_CHECK(k_dim >= 128 && k_dim % 128 == 0, "grouped_gemm_fp4: K %d must be a multiple of 128", k_dim);
    EXP_CHECK(n_dim >= 128 && n_dim % (swiglu ? 256 : 128) == 0, "grouped_gemm_fp4: N %d must be a multiple of %d", n_dim, swiglu ? 256 : 128);
    EXP_CHECK(static_cast<int64_t>(num_experts) * n_dim < (1ll << 31), "grouped_gemm_fp4: weight rows overflow");
    EXP_CHECK(aligned(a_s, 4) && aligned(w_s, 4), "grouped_gemm_fp4: scales must be 4-byte aligned");
    cam::GroupedGemmFp4Params p{};
    p.expert_offsets = offsets;
    p.num_experts = num_experts;
    p.rows = rows;
    p.n_dim = n_dim;
    p.k_dim = k_dim;
    p.a_scales = static_cast<const uint8_t*>(a_s);
    p.b_scales = static_cast<const uint8_t*>(w_s);
    p.scale_vec = k_dim % 256 == 0 && aligned(a_s, 16) && aligned(w_s, 16);
    p.a_gscale = a_gscale;
    p.b_gscale = w_gscale;
    p.out_gscale = out_gscale;
    p.out = out;
    p.out_scales = static_cast<uint8_t*>(out_s);
    CUtensorMap ta, ta32, tb;
    const uint64_t bytes = static_cast<uint64_t>(k_dim) / 2;
    if (map_2d(&ta, a_q, bytes, static_cast<uint64_t>(rows), 128) != 0) return -1;
    if (map_2d(&ta32, a_q, bytes, static_cast<uint64_t>(rows), 32) != 0) return -1;
    if (map_2d(&tb, w_q, bytes, static_cast<uint64_t>(num_experts) * n_dim, 128) != 0) return -1;
    return launched(cam_launch_grouped_gemm_fp4(&p, fmt, swiglu, &ta, &ta32, &tb, stream), "grouped_gemm_fp4");
}

extern "C" int cam_expert_ops_status(CamStatus* out) {
    const int rc = cam_fp4_status(out);
    return rc == 0 ? 0 : refuse("expert_ops_status: %s", cudaGetErrorString(static_cast<cudaError_t>(rc)));
}
