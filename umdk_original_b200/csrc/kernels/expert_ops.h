// Parameter blocks and C launchers of the expert-MLP operators that stand alone, without a Buffer: 4-bit quantisation,
// grouped products of 4-bit operands, grouped gated feed-forward in 16 bits with its backward pass.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../common/cam_types.h"

namespace cam {

// Programmatic dependent launch.  The kernels of these operators follow one another closely (quantise, gate and up, down; the
// products of a backward pass), each takes microseconds, and the start of one (launch, barriers, tensor memory) can overlap the
// end of the one before: a kernel waits for its predecessor's results only before its first access to memory (pdl_wait), and
// allows its successor to start once it runs itself (pdl_release).
#ifdef __CUDACC__
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
#endif
inline cudaLaunchAttribute pdl_attribute() {
    cudaLaunchAttribute a = {};
    a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a.val.programmaticStreamSerializationAllowed = 1;
    return a;
}

constexpr int kDtBf16 = 0, kDtFp16 = 1, kDtFp32 = 2;

struct GroupedGemmFp4Params {
    CamStatus* status;          // where a wait that ran out is recorded (host memory)
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

// Products of the gated feed-forward block in 16 bits (grouped_mlp.cu)
constexpr int kMlpUp = 0, kMlpDown = 1, kMlpDact = 2, kMlpDx = 3, kMlpDw = 4;

struct GroupedMlpParams {
    CamStatus* status;          // where a wait that ran out is recorded (host memory)
    const int* expert_offsets;  // [E+1]
    int num_experts, rows;      // rows of the row operands
    int m_dim;                  // kMlpDw: rows of an expert's gradient
    int n_dim;                  // columns of the result (I for kMlpUp and kMlpDact)
    int k_dim;                  // contraction (not kMlpDw)
    int fp16;                   // operands and results are fp16, otherwise bf16
    void* out;                  // [rows, n_dim]; kMlpDact: dgu [rows, 2 n_dim]; kMlpDw: [E, m_dim, n_dim]
    float* gate_up;             // [rows, 2I] fp32: written by kMlpUp (or null), read by kMlpDact
};

constexpr int kGvMaxSmem = 96 * 1024;  // shared memory of the form on the ordinary cores (expert_gemv.cu): up to four rows

// Form of the row products for experts with few rows (expert_gemm_narrow.cu): tiles of 128 weight rows x slot_rows rows.
constexpr int kNarrow16 = 2;  // beside the formats of fp4.cuh: 16-bit operands
// Weights contracted over their columns, plain or with SwiGLU; over their rows (16 bits): the gradient of the activation, or plain
constexpr int kNarrowPlain = 0, kNarrowSwiglu = 1, kNarrowDact = 2, kNarrowByRows = 3;
struct NarrowParams {
    CamStatus* status;          // where a wait that ran out is recorded (host memory)
    const int* expert_offsets;
    int num_experts, rows;
    int n_dim;                  // columns of the result; with SwiGLU: I, the weights have 2I rows
    int kblocks;                // 128-byte blocks of a row
    int slot_rows;              // rows of a tile at most: 32, 64 or 128
    int split;                  // CTAs of a cluster that share the K-blocks of a tile: 1, 2 or 4
    int chunks;                 // K-blocks of a stage: 1 or 2
    int chunked;                // the maps split rows into 128-byte K-blocks (rows of whole blocks only; needed for 2 chunks)
    int stages, stage_bytes;
    int fp16;
    void* out;                  // 16-bit [rows, n_dim], or fp4 SwiGLU: codes [rows, I/2]
    float* gate_up;             // 16-bit SwiGLU: null or fp32 [rows, 2I]; kNarrowDact: read
    // fp4
    const uint8_t *a_scales, *b_scales;
    int scale_pitch, scale_vec;
    const float *a_gscale, *b_gscale, *out_gscale;
    uint8_t* out_scales;
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
// tmap_a: boxes of 128 rows, tmap_a32: of 32 rows, both on A [rows, K / 2 bytes]; tmap_b: boxes of 128 rows on W [E N, K / 2];
// tmap_out (not with SwiGLU, where any map does): boxes of 32 rows on the result [rows, 2 N bytes]
int cam_launch_grouped_gemm_fp4(const cam::GroupedGemmFp4Params* p, int fmt, int swiglu, const CUtensorMap* tmap_a,
                                const CUtensorMap* tmap_a32, const CUtensorMap* tmap_b, const CUtensorMap* tmap_out, cudaStream_t stream);
// tmap_a: the row operand in boxes of 128 rows (kMlpDw: 64 rows), tmap_a32: in boxes of 32 rows; tmap_b: the weights
// [E, rows, columns] in boxes of 128 rows, or of 64 where their row is the contraction index (kMlpDact, kMlpDx), or for kMlpDw
// the second row operand in boxes of 64 rows.  tmap_out: the result in boxes of 32 rows, as [rows, 2, I] for kMlpDact, or [E, m_dim,
// n_dim] in boxes of 128 rows (kMlpDw).  All boxes are 128 bytes wide.  Not used, any map does: tmap_a32 of kMlpDw.
int cam_launch_grouped_mlp(const cam::GroupedMlpParams* p, int form, const CUtensorMap* tmap_a, const CUtensorMap* tmap_a32,
                           const CUtensorMap* tmap_b, const CUtensorMap* tmap_out, cudaStream_t stream);
// kind: kFp4Nv, kFp4Mx or kNarrow16.  The maps, innermost first; with `chunked` a row is (K-block, 128 bytes), otherwise all of
// its bytes and one K-block: tmap_a {bytes, rows, K-blocks} in boxes {128, slot_rows (32 without chunks), chunks}; tmap_b {bytes,
// rows, halves, K-blocks, experts} in boxes {128, 128 / halves, halves, chunks, 1} with SwiGLU's gate and up rows as two halves, or, for
// weights contracted over their rows, {bytes, rows, experts} in boxes {128, 64, 1}.
int cam_launch_expert_gemm_narrow(const cam::NarrowParams* p, int kind, int form, int64_t tiles, const CUtensorMap* tmap_a,
                                  const CUtensorMap* tmap_b, cudaStream_t stream);
// up and down (kMlpUp, kMlpDown) of a handful of rows; x and w 16-byte aligned
int cam_launch_expert_gemv(const cam::GroupedMlpParams* p, int swiglu, const void* x, const void* w, cudaStream_t stream);
int cam_expert_narrow_max_stages(void);
int cam_expert_narrow_fixed_smem(int fp4, int slot_rows);  // shared memory beside the stages
}
