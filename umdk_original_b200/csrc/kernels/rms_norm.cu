// rms_norm / add_rms_norm, the same with rows in 8 bits, and their backward pass.
//
//   s = x + residual (rounded to the residual's type),  r = 1 / sqrt(mean(s^2) + eps),  y = s r w
//   dx = dresidual = ds + r (w dy - s r mean(w dy s r)),   dw = sum over the rows of dy s r
//
// Bound by memory in both directions.  A row stays in the registers of the threads that share it: read once, summed, scaled and
// written.  Rows of up to 1024 values belong to one warp, longer ones to a block.  The norm is that of the rounded sum, so a
// backward pass (or a later layer) that reads the stored sum sees the numbers that were normalised.
#include "../common/quant.cuh"
#include "layer_ops.h"
#include "layer_values.cuh"
#include "launch.h"

namespace cam {

namespace {

constexpr int kRowsOnly = 0, kInt8 = 2, kE4m3 = 3;
constexpr int kWarpRows = 8;  // rows of a block where a row belongs to a warp

// Places of a thread's values: with VEC pieces of eight consecutive ones, otherwise (odd widths, any alignment) single ones.
template <bool VEC>
__device__ __forceinline__ int place(int v, int j, int t, int threads) {
    return VEC ? (v * threads + t) * 8 + j : (v * 8 + j) * threads + t;
}

template <int DT, bool VEC>
__device__ __forceinline__ void load_piece(const void* base, int64_t row0, int v, int t, int threads, int h, float* f) {
    if constexpr (VEC) {
        const int c = place<true>(v, 0, t, threads);
        if (c < h) widen8<DT>(load8<DT>(base, row0 + c), f);
        else {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = 0.f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = place<false>(v, j, t, threads);
            f[j] = c < h ? load1<DT>(base, row0 + c) : 0.f;
        }
    }
}

template <int DT, bool VEC>
__device__ __forceinline__ void store_piece(void* base, int64_t row0, int v, int t, int threads, int h, const float* f) {
    if constexpr (VEC) {
        const int c = place<true>(v, 0, t, threads);
        if (c < h) store8<DT>(base, row0 + c, narrow8<DT>(f));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = place<false>(v, j, t, threads);
            if (c < h) store1<DT>(base, row0 + c, f[j]);
        }
    }
}

// Weights are read by every row: through L1.
template <int DT, bool VEC>
__device__ __forceinline__ void load_weight(const void* w, bool fp32, int v, int t, int threads, int h, float* f) {
    if constexpr (VEC) {
        const int c = place<true>(v, 0, t, threads);
        if (c >= h) {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = 0.f;
        } else if (fp32 || DT == kDtFp32) {
            const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(w) + c);
            const float4 a = __ldg(p), b = __ldg(p + 1);
            f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
        } else if constexpr (DT != kDtFp32) {
            Raw8<DT> r;
            r.v[0] = __ldg(reinterpret_cast<const uint4*>(static_cast<const char*>(w) + c * 2));
            widen8<DT>(r, f);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = place<false>(v, j, t, threads);
            f[j] = c >= h ? 0.f : fp32 ? load1<kDtFp32>(w, c) : load1<DT>(w, c);
        }
    }
}

// Sum (and maximum) over the threads that share a row; `red`: 64 floats of the block.
template <bool WARP, bool MAX>
__device__ __forceinline__ void over_row(float& sum, float& top, float* red) {
    sum = warp_sum(sum);
    if (MAX) top = warp_max(top);
    if constexpr (!WARP) {
        const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
        __syncthreads();  // the row before has been read from `red`
        if (lane == 0) {
            red[threadIdx.x >> 5] = sum;
            if (MAX) red[32 + (threadIdx.x >> 5)] = top;
        }
        __syncthreads();
        sum = warp_sum(lane < warps ? red[lane] : 0.f);
        if (MAX) top = warp_max(lane < warps ? red[32 + lane] : 0.f);
    }
}

// Threads of a block at most: four pieces per thread up to 8192 values, two beyond
constexpr int norm_threads(int pieces, bool warp) { return warp || pieces == 4 ? 256 : 1024; }
static_assert(kWarpRows * 32 == 256 && 256 * 4 * 8 >= 8192 && 1024 * 2 * 8 >= kNormMaxHidden, "every row has its threads");

template <int DT, int MODE, int NV, bool VEC, bool WARP>
__global__ void __launch_bounds__(norm_threads(NV, WARP))
rms_norm_kernel(const RmsNormParams p) {
    __shared__ float red[64];
    const int threads = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
    const int h = p.h;
    const int64_t row0 = row * h;
    pdl_wait();
    pdl_release();
    if (WARP && row >= p.rows) return;
    float s[NV * 8], w[NV * 8];
#pragma unroll
    for (int v = 0; v < NV; ++v) load_piece<DT, VEC>(p.x, row0, v, t, threads, h, s + 8 * v);
    if (p.residual != nullptr) {
        if (DT == kDtFp32 || p.res_type == kDtFp32) {
#pragma unroll
            for (int v = 0; v < NV; ++v) load_piece<kDtFp32, VEC>(p.residual, row0, v, t, threads, h, w + 8 * v);
#pragma unroll
            for (int i = 0; i < NV * 8; ++i) s[i] += w[i];
#pragma unroll
            for (int v = 0; v < NV; ++v) store_piece<kDtFp32, VEC>(p.sum, row0, v, t, threads, h, s + 8 * v);
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v) load_piece<DT, VEC>(p.residual, row0, v, t, threads, h, w + 8 * v);
#pragma unroll
            for (int i = 0; i < NV * 8; ++i) s[i] = rounded<DT>(s[i] + w[i]);
#pragma unroll
            for (int v = 0; v < NV; ++v) store_piece<DT, VEC>(p.sum, row0, v, t, threads, h, s + 8 * v);
        }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) load_weight<DT, VEC>(p.weight, p.weight_type == kDtFp32, v, t, threads, h, w + 8 * v);
    float sum = 0.f, top = 0.f;
#pragma unroll
    for (int i = 0; i < NV * 8; ++i) {
        sum = fmaf(s[i], s[i], sum);
        if (MODE == kInt8) top = fmaxf(top, fabsf(s[i] * w[i]));
    }
    over_row<WARP, MODE == kInt8>(sum, top, red);
    const float rstd = 1.f / sqrtf(sum / static_cast<float>(h) + p.eps);
    if (p.rstd != nullptr && t == 0) p.rstd[row] = rstd;
#pragma unroll
    for (int i = 0; i < NV * 8; ++i) s[i] = s[i] * rstd * w[i];
    if (MODE == kRowsOnly || p.y != nullptr) {
#pragma unroll
        for (int v = 0; v < NV; ++v) store_piece<DT, VEC>(p.y, row0, v, t, threads, h, s + 8 * v);
    }
    if constexpr (MODE == kInt8) {
        // a row with NaN has a NaN scale
        const float inv = 127.f / (top * rstd + 1e-12f);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            int q[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = max(-127, min(127, __float2int_rn(s[8 * v + j] * inv)));
            if constexpr (VEC) {
                const int c = place<true>(v, 0, t, threads);
                uint2 o = make_uint2(0u, 0u);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    o.x |= (static_cast<uint32_t>(q[j]) & 0xFFu) << (8 * j);
                    o.y |= (static_cast<uint32_t>(q[4 + j]) & 0xFFu) << (8 * j);
                }
                if (c < h) *reinterpret_cast<uint2*>(static_cast<int8_t*>(p.q) + row0 + c) = o;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int c = place<false>(v, j, t, threads);
                    if (c < h) static_cast<int8_t*>(p.q)[row0 + c] = static_cast<int8_t>(q[j]);
                }
            }
        }
        if (t == 0) p.scales[row] = 1.f / inv;
    }
    if constexpr (MODE == kE4m3) {
        // a block of 128 values: sixteen consecutive lanes
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float* f = s + 8 * v;
            float amax = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(f[j]));
#pragma unroll
            for (int o = 8; o >= 1; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
            float scale, inv;
            if (p.quant_mode == 4) ue8m0_scale(amax, scale, inv);
            else {
                const float a = fmaxf(amax, 1e-4f);
                inv = 448.f / a;
                scale = a / 448.f;
            }
            const int c = place<true>(v, 0, t, threads);
            if (c < h) {
                *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.q) + row0 + c) =
                    make_uint2(pack_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv), pack_e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
                if ((t & 15) == 0) p.scales[row * (h / 128) + (c >> 7)] = scale;
            }
        }
    }
}

// Rows are shared out to the blocks in turn; a thread keeps the sums of its columns' weight gradients over all of its rows, and the
// block's go to `partial`, which a second kernel adds up in a fixed order.
template <int DT, int NV, bool VEC, bool WARP, int THREADS>
__global__ void __launch_bounds__(THREADS)
rms_norm_backward_kernel(const RmsNormBackwardParams p) {
    __shared__ float red[64];
    __shared__ float cols[WARP ? kWarpRows * NV * 256 : 1];
    const int threads = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x, warp = threadIdx.x >> 5;
    const int h = p.h;
    const int64_t first = WARP ? static_cast<int64_t>(blockIdx.x) * kWarpRows + warp : blockIdx.x;
    const int64_t step = WARP ? static_cast<int64_t>(gridDim.x) * kWarpRows : gridDim.x;
    const bool sum32 = DT == kDtFp32 || p.sum_type == kDtFp32;
    pdl_wait();
    pdl_release();
    float w[NV * 8], acc[NV * 8];
#pragma unroll
    for (int v = 0; v < NV; ++v) load_weight<DT, VEC>(p.weight, p.weight_type == kDtFp32, v, t, threads, h, w + 8 * v);
#pragma unroll
    for (int i = 0; i < NV * 8; ++i) acc[i] = 0.f;
    for (int64_t row = first; row < p.rows; row += step) {
        const int64_t row0 = row * h;
        float dy[NV * 8], hat[NV * 8], ds[NV * 8];
#pragma unroll
        for (int v = 0; v < NV; ++v) load_piece<DT, VEC>(p.dy, row0, v, t, threads, h, dy + 8 * v);
        if (sum32) {
#pragma unroll
            for (int v = 0; v < NV; ++v) load_piece<kDtFp32, VEC>(p.sum, row0, v, t, threads, h, hat + 8 * v);
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v) load_piece<DT, VEC>(p.sum, row0, v, t, threads, h, hat + 8 * v);
        }
        if (p.dsum == nullptr) {
#pragma unroll
            for (int i = 0; i < NV * 8; ++i) ds[i] = 0.f;
        } else if (sum32) {
#pragma unroll
            for (int v = 0; v < NV; ++v) load_piece<kDtFp32, VEC>(p.dsum, row0, v, t, threads, h, ds + 8 * v);
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v) load_piece<DT, VEC>(p.dsum, row0, v, t, threads, h, ds + 8 * v);
        }
        const float rstd = __ldg(p.rstd + row);
        float along = 0.f, none = 0.f;
#pragma unroll
        for (int i = 0; i < NV * 8; ++i) {
            hat[i] *= rstd;
            acc[i] = fmaf(dy[i], hat[i], acc[i]);
            dy[i] *= w[i];
            along = fmaf(dy[i], hat[i], along);
        }
        over_row<WARP, false>(along, none, red);
        along /= static_cast<float>(h);
#pragma unroll
        for (int i = 0; i < NV * 8; ++i) ds[i] = fmaf(rstd, fmaf(-along, hat[i], dy[i]), ds[i]);
        if (p.dx != nullptr) {
#pragma unroll
            for (int v = 0; v < NV; ++v) store_piece<DT, VEC>(p.dx, row0, v, t, threads, h, ds + 8 * v);
        }
        if (p.dres != nullptr) {
            if (sum32) {
#pragma unroll
                for (int v = 0; v < NV; ++v) store_piece<kDtFp32, VEC>(p.dres, row0, v, t, threads, h, ds + 8 * v);
            } else {
#pragma unroll
                for (int v = 0; v < NV; ++v) store_piece<DT, VEC>(p.dres, row0, v, t, threads, h, ds + 8 * v);
            }
        }
    }
    if (p.partial == nullptr) return;
    float* mine = p.partial + static_cast<int64_t>(blockIdx.x) * h;
    if constexpr (WARP) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int c = place<VEC>(v, j, t, threads);
                if (c < h) cols[warp * NV * 256 + c] = acc[8 * v + j];
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < h; c += blockDim.x) {
            float a = 0.f;
#pragma unroll
            for (int r = 0; r < kWarpRows; ++r) a += cols[r * NV * 256 + c];
            mine[c] = a;
        }
    } else {
#pragma unroll
        for (int v = 0; v < NV; ++v) store_piece<kDtFp32, VEC>(mine, 0, v, t, threads, h, acc + 8 * v);
    }
}

// dw[c] = sum over the parts: 32 columns and 8 shares of the parts per block
template <int DT>
__global__ void __launch_bounds__(256) add_parts_kernel(const float* __restrict__ partial, int parts, int h, void* dw) {
    __shared__ float red[8][33];
    const int lane = threadIdx.x & 31, share = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    pdl_wait();
    pdl_release();
    float a = 0.f;
    if (c < h) {
#pragma unroll 8
        for (int i = share; i < parts; i += 8) a += __ldg(partial + static_cast<int64_t>(i) * h + c);
    }
    red[share][lane] = a;
    __syncthreads();
    if (share == 0 && c < h) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += red[i][lane];
        store1<DT>(dw, c, sum);
    }
}

// Threads that share a row and pieces of eight values per thread
struct Shape {
    bool warp;
    int threads, pieces;
};

Shape shape_of(int h, int warp_pieces, int block_pieces) {
    const int pieces = (h + 7) / 8;
    if (pieces <= 32 * warp_pieces) {
        const int per = (pieces + 31) / 32;
        return {true, kWarpRows * 32, per <= 1 ? 1 : per <= 2 ? 2 : 4};
    }
    const int threads = ((pieces + block_pieces - 1) / block_pieces + 31) / 32 * 32;
    return {false, threads, block_pieces};
}

template <int DT, int MODE, int NV, bool VEC>
int launch_norm(const RmsNormParams& p, const Shape& s, cudaStream_t stream) {
    if (s.warp)
        return launch_pdl(rms_norm_kernel<DT, MODE, NV, VEC, true>, dim3(static_cast<unsigned>((p.rows + kWarpRows - 1) / kWarpRows)), s.threads, 0, stream, p);
    if constexpr (NV >= 2) return launch_pdl(rms_norm_kernel<DT, MODE, NV, VEC, false>, dim3(static_cast<unsigned>(p.rows)), s.threads, 0, stream, p);
    return static_cast<int>(cudaErrorInvalidValue);
}

template <int DT, int MODE, bool VEC>
int launch_norm_pieces(const RmsNormParams& p, cudaStream_t stream) {
    const Shape s = shape_of(p.h, 4, p.h > 8192 ? 2 : 4);
    if (s.pieces == 1) return launch_norm<DT, MODE, 1, VEC>(p, s, stream);
    if (s.pieces == 2) return launch_norm<DT, MODE, 2, VEC>(p, s, stream);
    return launch_norm<DT, MODE, 4, VEC>(p, s, stream);
}

template <int DT>
int launch_norm_type(const RmsNormParams& p, cudaStream_t stream) {
    const bool vec = p.h % 8 == 0 && aligned16(p.x) && aligned16(p.residual) && aligned16(p.weight) && aligned16(p.y) && aligned16(p.sum) && aligned16(p.q);
    if (p.quant_mode == 0) return vec ? launch_norm_pieces<DT, kRowsOnly, true>(p, stream) : launch_norm_pieces<DT, kRowsOnly, false>(p, stream);
    if (p.quant_mode == 2) return vec ? launch_norm_pieces<DT, kInt8, true>(p, stream) : launch_norm_pieces<DT, kInt8, false>(p, stream);
    return vec && p.h % 128 == 0 ? launch_norm_pieces<DT, kE4m3, true>(p, stream) : static_cast<int>(cudaErrorInvalidValue);
}

Shape backward_shape(int h) { return shape_of(h, 2, 2); }

template <int DT, int NV, bool VEC>
int launch_backward(const RmsNormBackwardParams& p, const Shape& s, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>(p.parts));
    if (s.warp) return launch_pdl(rms_norm_backward_kernel<DT, NV, VEC, true, kWarpRows * 32>, grid, s.threads, 0, stream, p);
    if constexpr (NV == 2) {
        if (s.threads <= 512) return launch_pdl(rms_norm_backward_kernel<DT, 2, VEC, false, 512>, grid, s.threads, 0, stream, p);
        return launch_pdl(rms_norm_backward_kernel<DT, 2, VEC, false, 1024>, grid, s.threads, 0, stream, p);
    }
    return static_cast<int>(cudaErrorInvalidValue);
}

template <int DT>
int launch_backward_type(const RmsNormBackwardParams& p, cudaStream_t stream) {
    const bool vec = p.h % 8 == 0 && aligned16(p.dy) && aligned16(p.dsum) && aligned16(p.sum) && aligned16(p.weight) && aligned16(p.dx) &&
                     aligned16(p.dres) && aligned16(p.partial);
    const Shape s = backward_shape(p.h);
    int rc;
    if (s.pieces == 1) rc = vec ? launch_backward<DT, 1, true>(p, s, stream) : launch_backward<DT, 1, false>(p, s, stream);
    else rc = vec ? launch_backward<DT, 2, true>(p, s, stream) : launch_backward<DT, 2, false>(p, s, stream);
    if (rc != 0 || p.dweight == nullptr) return rc;
    auto add = p.weight_type == kDtFp32 ? add_parts_kernel<kDtFp32> : p.weight_type == kDtFp16 ? add_parts_kernel<kDtFp16> : add_parts_kernel<kDtBf16>;
    return launch_pdl(add, dim3(static_cast<unsigned>((p.h + 31) / 32)), 256, 0, stream, static_cast<const float*>(p.partial), p.parts, p.h, p.dweight);
}

}  // namespace

}  // namespace cam

extern "C" int cam_launch_rms_norm(const cam::RmsNormParams* p, int dtype, cudaStream_t stream) {
    using namespace cam;
    return dtype == kDtBf16 ? launch_norm_type<kDtBf16>(*p, stream) : dtype == kDtFp16 ? launch_norm_type<kDtFp16>(*p, stream) : launch_norm_type<kDtFp32>(*p, stream);
}

extern "C" int cam_rms_norm_backward_blocks(int64_t rows, int h) {
    using namespace cam;
    const Shape s = backward_shape(h);
    const int64_t turns = s.warp ? (rows + kWarpRows - 1) / kWarpRows : rows;
    const int64_t most = static_cast<int64_t>(sm_count_of_current_device()) * (s.threads <= 512 ? 2 : 1);
    return static_cast<int>(turns < most ? turns : most);
}

extern "C" int cam_launch_rms_norm_backward(const cam::RmsNormBackwardParams* p, int dtype, cudaStream_t stream) {
    using namespace cam;
    return dtype == kDtBf16 ? launch_backward_type<kDtBf16>(*p, stream) : dtype == kDtFp16 ? launch_backward_type<kDtFp16>(*p, stream) : launch_backward_type<kDtFp32>(*p, stream);
}
