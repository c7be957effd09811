// C interface of the expert-MLP operators that need no Buffer.  Like cam_runtime.h: no PyTorch, raw device pointers, 0 on
// success and cam_last_error() otherwise.  The products write to one page of host memory, allocated by the first of them; nothing else
// allocates, and only cam_expert_ops_status waits.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../common/cam_types.h"

#ifdef __cplusplus
extern "C" {
#endif

// dtype: 0 bf16, 1 fp16, 2 fp32.  fmt: 0 nvfp4 (e4m3 scale per 16 values), 1 mxfp4 (e8m0 scale per 32).
// numel is a multiple of the block; gscale: null, or `gscales` floats that each cover numel / gscales values (nvfp4 only).
int cam_quantize_fp4(const void* x, int dtype, int fmt, void* q, void* s, int64_t numel, const float* gscale, int64_t gscales,
                     cudaStream_t stream);
int cam_dequantize_fp4(const void* q, const void* s, int dtype, int fmt, void* out, int64_t numel, const float* gscale,
                       int64_t gscales, cudaStream_t stream);

// a_q [rows, K/2], a_s [rows, K/block], w_q [E, N, K/2], w_s [E, N, K/block], offsets int32 [E+1] on the device.
// swiglu 0: out bf16 [rows, N].  swiglu 1: N = 2I (gate rows first), out codes [rows, I/2], out_s [rows, I/block].
// Rows outside [offsets[0], offsets[E]) are written as zeros.
int cam_grouped_gemm_fp4(const void* a_q, const void* a_s, int rows, const void* w_q, const void* w_s, const int* offsets,
                         int num_experts, int n_dim, int k_dim, int fmt, int swiglu, const float* a_gscale,
                         const float* w_gscale, const float* out_gscale, void* out, void* out_s, cudaStream_t stream);

// Gated feed-forward block of 16-bit experts (kernels/grouped_mlp.cu), dtype 0 bf16 or 1 fp16.  x, y, dy, dx [rows, h], w1, dw1
// [E, 2I, h] (gate rows first), w2, dw2 [E, h, I], act [rows, I]; gate_up [rows, 2I] fp32 (null: not kept), dgu [rows, 2I].
// Rows outside [offsets[0], offsets[E]) of y and dx, and gradients of experts without rows, are written as zeros.
int cam_grouped_mlp_up(const void* x, const void* w1, const int* offsets, int rows, int num_experts, int h, int inter, int dtype,
                       void* act, float* gate_up, cudaStream_t stream);
int cam_grouped_mlp_down(const void* act, const void* w2, const int* offsets, int rows, int num_experts, int h, int inter, int dtype,
                         void* y, cudaStream_t stream);
int cam_grouped_mlp_dact(const void* dy, const void* w2, const float* gate_up, const int* offsets, int rows, int num_experts, int h,
                         int inter, int dtype, void* dgu, cudaStream_t stream);
int cam_grouped_mlp_dx(const void* dgu, const void* w1, const int* offsets, int rows, int num_experts, int h, int inter, int dtype,
                       void* dx, cudaStream_t stream);
// dw[e] = a[rows of e]^T b[rows of e]: a [rows, m_dim], b [rows, n_dim], dw [E, m_dim, n_dim]
int cam_grouped_mlp_dw(const void* a, const void* b, const int* offsets, int rows, int num_experts, int m_dim, int n_dim, int dtype,
                       void* dw, cudaStream_t stream);

// A wait inside a product that ran out on the current device (code 0: none); waits for the device, and clears it where asked to.
// Until it is cleared every further product on that device is refused.  cam_expert_ops_set_status is for tests of the host's side.
int cam_expert_ops_status(CamStatus* out, int clear);
int cam_expert_ops_set_status(const CamStatus* st);

#ifdef __cplusplus
}
#endif
