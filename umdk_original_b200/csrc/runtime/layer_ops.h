// C interface of the operators round the experts: residual and norm, routing, rows grouped by expert and brought back.  Like
// expert_ops.h: raw device pointers, no PyTorch, 0 on success and cam_last_error() otherwise; nothing allocates or waits.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

// dtype (of x, y), res_type (of residual, sum: dtype or fp32), weight_type: 0 bf16, 1 fp16, 2 fp32.  residual null: no sum.  y null with a
// quant mode only.  rstd [rows] or null.  quant_mode 0: none; 2: q int8 [rows, h], scales [rows]; 3, 4: q e4m3, scales [rows, h / 128],
// fp32 or powers of two (h a multiple of 128, 16-byte aligned).
int cam_rms_norm(const void* x, int dtype, const void* residual, int res_type, const void* weight, int weight_type, int64_t rows, int h,
                 float eps, void* y, void* sum, float* rstd, int quant_mode, void* q, float* scales, cudaStream_t stream);
// Rows of the workspace `partial` [parts, h] fp32 that a gradient of the weight needs
int cam_rms_norm_backward_parts(int64_t rows, int h);
// dy, dx of dtype; dsum (or null), sum, dres of sum_type; outputs that are null are left out
int cam_rms_norm_backward(const void* dy, int dtype, const void* dsum, const void* sum, int sum_type, const void* weight, int weight_type,
                          const float* rstd, int64_t rows, int h, void* dx, void* dres, void* dweight, float* partial, int parts,
                          cudaStream_t stream);

// logits [rows, experts]; bias fp32 [experts] or null; idx int64 [rows, k], weights fp32 [rows, k]
int cam_moe_route(const void* logits, int dtype, int64_t rows, int experts, int k, const float* bias, int sigmoid, int groups,
                  int topk_groups, int group_top, int renormalize, float scale, int64_t* idx, float* weights, cudaStream_t stream);
int cam_moe_route_backward(const float* dweights, const void* logits, int dtype, const int64_t* idx, int64_t rows, int experts, int k,
                           int sigmoid, int renormalize, float scale, void* dlogits, cudaStream_t stream);

// x [tokens, row_bytes] of elements of 1, 2 or 4 bytes, scales [tokens, scale_cols] or null, idx [tokens, k] int32 / int64 -> rows [tokens * k, row_bytes], row_scales,
// offsets int32 [experts + 1], slots int32 [tokens, k] (-1: the id is outside [0, experts)); rows past offsets[experts] are zeros
int cam_moe_group_rows(const void* x, int64_t row_bytes, int elem_bytes, const float* scales, int scale_cols, const void* idx, int idx_i64, int64_t tokens,
                       int k, int experts, void* rows, float* row_scales, int* offsets, int* slots, cudaStream_t stream);
// out[t] = residual[t] + sum_j weights[t, j] rows[slots[t, j]]; slots outside [0, num_rows) add nothing
int cam_moe_ungroup_rows(const void* rows, int dtype, int64_t num_rows, int h, const int* slots, int64_t tokens, int k, const float* weights,
                         const void* residual, void* out, cudaStream_t stream);
// 32-bit words of the workspace `used` that gradients of rows need; 0: none
int64_t cam_moe_ungroup_rows_backward_words(int dtype, int64_t num_rows, int h, int64_t tokens, int k);
// A row belongs to one slot at most; rows of no slot get zeros.
int cam_moe_ungroup_rows_backward(const void* dout, const void* rows, int dtype, int64_t num_rows, int h, const int* slots, int64_t tokens,
                                  int k, const float* weights, void* drows, float* dweights, uint32_t* used, cudaStream_t stream);

#ifdef __cplusplus
}
#endif
