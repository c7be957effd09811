// Parameter blocks and C launchers of the operators round the experts: residual and norm, routing, rows grouped by expert.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "expert_ops.h"

namespace cam {

constexpr int kNormMaxHidden = 16384;   // 1024 threads x 16 values
constexpr int kRouteMaxExperts = 1024;  // 32 lanes x 32 values
constexpr int kLayerMaxTopk = 32;       // choices of a token

struct RmsNormParams {
    const void* x;          // [rows, h]
    const void* residual;   // [rows, h] of type res_type, or null
    const void* weight;     // [h] of type weight_type
    int res_type, weight_type;
    int64_t rows;
    int h;
    float eps;
    void* y;                // [rows, h] of x's type, or null
    void* sum;              // with a residual: [rows, h] of res_type
    float* rstd;            // [rows] or null
    int quant_mode;         // 0: none
    void* q;                // [rows, h]
    float* scales;          // [rows] (mode 2) or [rows, h / 128]
};

struct RmsNormBackwardParams {
    const void* dy;         // [rows, h]
    const void* dsum;       // [rows, h] of sum_type, or null
    const void* sum;        // [rows, h] of sum_type
    const void* weight;
    const float* rstd;
    int sum_type, weight_type;
    int64_t rows;
    int h;
    void* dx;               // [rows, h] of dy's type, or null
    void* dres;             // [rows, h] of sum_type, or null
    void* dweight;          // [h] of weight_type, or null
    float* partial;         // [parts, h], with dweight
    int parts;              // blocks that the rows are shared out to
};

struct RouteParams {
    const void* logits;     // [rows, experts]
    const float* bias;      // [experts] or null
    int64_t rows;
    int experts, k, groups, topk_groups, group_top, sigmoid, renormalize;
    float scale;
    int vec, vec_bias;      // a lane's logits and biases can be read in whole pieces (set by the launcher)
    int64_t* idx;           // [rows, k]
    float* weights;         // [rows, k]
    const float* dweights;  // backward
    void* dlogits;          // [rows, experts]
};

struct GroupRowsParams {
    const void* x;          // [tokens, row_bytes]
    const float* scales;    // [tokens, scale_cols] or null
    const void* idx;        // [tokens, k]
    int idx_i64;
    int64_t tokens;
    int k, experts, scale_cols;
    int64_t row_bytes;
    int elem_bytes;         // 1, 2 or 4
    void* rows;             // [tokens * k, row_bytes]
    float* row_scales;      // [tokens * k, scale_cols]
    int* offsets;           // [experts + 1]
    int* slots;             // [tokens, k]
};

struct UngroupRowsParams {
    const void* rows;       // [num_rows, h]
    int64_t num_rows;
    int h;
    const int* slots;       // [tokens, k]
    int64_t tokens;
    int k;
    const float* weights;   // [tokens, k] or null
    const void* residual;   // [tokens, h] or null
    void* out;              // [tokens, h]
    const void* dout;       // backward
    void* drows;            // [num_rows, h] or null
    float* dweights;        // [tokens, k] or null
    uint32_t* used;         // a bit per row, or null: workspace of gradients of many rows
};

}  // namespace cam

extern "C" {
int cam_launch_rms_norm(const cam::RmsNormParams* p, int dtype, cudaStream_t stream);
int cam_rms_norm_backward_blocks(int64_t rows, int h);
int cam_launch_rms_norm_backward(const cam::RmsNormBackwardParams* p, int dtype, cudaStream_t stream);
int cam_launch_moe_route(const cam::RouteParams* p, int dtype, cudaStream_t stream);
int cam_launch_group_rows(const cam::GroupRowsParams* p, cudaStream_t stream);
int cam_launch_ungroup_rows(const cam::UngroupRowsParams* p, int dtype, cudaStream_t stream);
int64_t cam_ungroup_rows_backward_map_words(int64_t num_rows, int h, int dtype, int64_t pairs);
int cam_launch_ungroup_rows_backward(const cam::UngroupRowsParams* p, int dtype, cudaStream_t stream);
}
