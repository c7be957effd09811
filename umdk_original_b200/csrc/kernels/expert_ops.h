// Parameter blocks and C launchers of the expert-MLP operators that stand alone, without a Buffer: 4-bit quantisation,
// grouped products of 4-bit operands, grouped gated feed-forward in 16 bits with its backward pass.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../common/cam_types.h"

namespace cam {

constexpr int kDtBf16 = 0, kDtFp16 = 1, kDtFp32 = 2;

struct GroupedGemmFp4Params {
    const int* expert_offsets;  // [E+1] first row of every expert
    int num_experts, rows;      // rows of A and of the outputs
    int n_dim, k_dim;           // N (2I for the SwiGLU form), K
    const uint8_t* a_scales;    // [rows, K / block]
    const uint8_t* b_scales;    // [E, N, K / block]
    int scale_vec;              // rows of both scale arrays can be read 16 (nvfp4) or 8 (mxfp4) bytes at a time
    const float* a_gscale;      // null or [1]
    const float* b_gscale;      // null or [E]
    const float* out_gscale;    // SwiGLU form: null or [1]
    void* out;                  // bf16 [rows, N], or the SwiGLU form's codes [rows, I / 2]
    uint8_t* out_scales;        // SwiGLU form: [rows, I / block]
};

}  // namespace cam

extern "C" {
// runtime/cam_runtime.cpp: a tensor map over bytes with 128-byte swizzle, zeros outside; dims and box innermost first, strides
// (bytes) of dimensions 1...; and the text that cam_last_error() returns next (returns -1)
int cam_encode_tmap(CUtensorMap* out, const void* base, int rank, const uint64_t* dims, const uint64_t* strides, const uint32_t* box);
int cam_fail(const char* message);
int cam_launch_quantize_fp4(const void* x, int dtype, int fmt, void* q, void* s, int64_t groups, const float* gscale,
                            int64_t groups_per_scale, cudaStream_t stream);
int cam_launch_dequantize_fp4(const void* q, const void* s, int dtype, int fmt, void* out, int64_t groups,
                              const float* gscale, int64_t groups_per_scale, cudaStream_t stream);
// tmap_a: boxes of 128 rows, tmap_a32: of 32 rows, both on A [rows, K / 2 bytes]; tmap_b: boxes of 128 rows on W [E N, K / 2]
int cam_launch_grouped_gemm_fp4(const cam::GroupedGemmFp4Params* p, int fmt, int swiglu, const CUtensorMap* tmap_a,
                                const CUtensorMap* tmap_a32, const CUtensorMap* tmap_b, cudaStream_t stream);
int cam_fp4_status(CamStatus* out);  // of the current device: the first wait that ran out in any grouped_gemm_fp4 kernel
}
