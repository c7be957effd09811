// Up (with SwiGLU) and down products of 16-bit experts for a handful of rows: every weight row is read once by one warp and
// multiplied on the ordinary cores.
//
// At so few rows nothing but the stream of weights counts, and the tensor core's forms pay for stages, accumulators and an exchange
// between CTAs that a call of ten microseconds does not earn back.  A warp owns two weight rows (the gate and the up row of a feature,
// or two neighbouring features); a lane reads 16 bytes of each at a time, four such steps ahead of the four it multiplies with up to four
// rows of the expert, which stay in shared memory.  The lanes' sums are added in a fixed order.  Sums are fp32; the products of two
// 16-bit values are exact in it.
// One row, 7168 x 2048 (88 MB of weights in two launches): 19.9 us, 4.4 TB/s, against 26.7 us on the tensor cores.  Without the loads
// ahead and with the rows from L1 it was 25.6 us.  Each further row costs 2 to 4 us of arithmetic: past three rows the tensor cores win.
#include "expert_gemm.cuh"

namespace cam {

constexpr int kGvThreads = 256, kGvWarps = kGvThreads / 32;
constexpr int kGvSteps = 4;  // 16-byte loads of each weight row in flight per lane

namespace {

template <bool FP16>
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (FP16) {
            const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = t.x;
            f[2 * i + 1] = t.y;
        } else {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
}
__device__ __forceinline__ uint4 load_once(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

}  // namespace

// R: rows of an expert that are taken at a time; their values stay in shared memory as [row][k].
template <bool SWIGLU, bool FP16, int R>
__global__ void __launch_bounds__(kGvThreads, 2)
expert_gemv_kernel(const uint4* __restrict__ x, const uint4* __restrict__ w, const GroupedMlpParams p) {
    extern __shared__ uint4 xs[];
    pdl_wait();
    pdl_release();
    const int warp = static_cast<int>(threadIdx.x) >> 5;
    const int lane = static_cast<int>(lane_id());
    constexpr int F = SWIGLU ? 1 : 2;  // result columns of a warp
    const int groups = (p.n_dim + F * kGvWarps - 1) / (F * kGvWarps);
    RowWalker<R> walker(p.expert_offsets, p.num_experts, groups, p.rows);
    int e, nt, row0, rows;
    if (walker.locate(static_cast<int>(blockIdx.x), e, nt, row0, rows)) {
        const int c = (nt * kGvWarps + warp) * F;  // n_dim is a multiple of 8: both columns exist or none
        const int pitch = p.k_dim / 8;             // 16-byte units of a row
        const bool live = c < p.n_dim;
        const uint4* w0 = w + (static_cast<size_t>(e) * (SWIGLU ? 2 * static_cast<size_t>(p.n_dim) : p.n_dim) + (live ? c : 0)) * pitch;
        const uint4* w1 = w0 + (SWIGLU ? static_cast<size_t>(p.n_dim) : 1) * pitch;
        uint4 a[kGvSteps], b[kGvSteps];
        auto load = [&](int k0) {
#pragma unroll
            for (int s = 0; s < kGvSteps; ++s) {
                const int k = k0 + 32 * s;
                a[s] = k < pitch ? load_once(w0 + k) : make_uint4(0, 0, 0, 0);
                b[s] = k < pitch ? load_once(w1 + k) : make_uint4(0, 0, 0, 0);
            }
        };
        load(lane);
        const uint4* xr = x + static_cast<size_t>(row0) * pitch;
        for (int i = static_cast<int>(threadIdx.x); i < rows * pitch; i += kGvThreads) xs[i] = __ldg(xr + i);
        __syncthreads();
        if (live) {
            float acc[2][R] = {};
            for (int k0 = lane; k0 < pitch; k0 += 32 * kGvSteps) {
                uint4 ca[kGvSteps], cb[kGvSteps];
#pragma unroll
                for (int s = 0; s < kGvSteps; ++s) {
                    ca[s] = a[s];
                    cb[s] = b[s];
                }
                load(k0 + 32 * kGvSteps);  // on their way while the present ones are multiplied
#pragma unroll
                for (int s = 0; s < kGvSteps; ++s) {
                    const int k = k0 + 32 * s;
                    if (k < pitch) {
                        float fa[8], fb[8];
                        unpack8<FP16>(ca[s], fa);
                        unpack8<FP16>(cb[s], fb);
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            if (r < rows) {
                                float fx[8];
                                unpack8<FP16>(xs[r * pitch + k], fx);
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    acc[0][r] = fmaf(fa[i], fx[i], acc[0][r]);
                                    acc[1][r] = fmaf(fb[i], fx[i], acc[1][r]);
                                }
                            }
                        }
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (r >= rows) break;
                float v[2] = {acc[0][r], acc[1][r]};
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) {
                    v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], d);
                    v[1] += __shfl_xor_sync(0xFFFFFFFFu, v[1], d);
                }
                if (lane == 0) {
                    const size_t row = static_cast<size_t>(row0 + r);
                    uint16_t* out = static_cast<uint16_t*>(p.out) + row * p.n_dim + c;
                    if constexpr (SWIGLU) {
                        if (p.gate_up != nullptr) {
                            float* gu = p.gate_up + row * (2 * static_cast<size_t>(p.n_dim)) + c;
                            gu[0] = v[0];
                            gu[p.n_dim] = v[1];
                        }
                        *out = static_cast<uint16_t>(pack16(v[0] * sigmoid_fast(v[0]) * v[1], 0.f, FP16));
                    } else {
                        *reinterpret_cast<uint32_t*>(out) = pack16(v[0], v[1], FP16);  // c is even
                    }
                }
            }
        }
    }
    zero_loose_rows(p.out, p.n_dim / 8, p.expert_offsets, p.num_experts, p.rows, static_cast<int>(threadIdx.x), kGvThreads);
}

}  // namespace cam

namespace {

template <bool SWIGLU, bool FP16, int R>
int launch_gemv(const cam::GroupedMlpParams* p, const void* x, const void* w, cudaStream_t stream) {
    static cam::SmemLimitCache limit;
    constexpr int columns = (SWIGLU ? 1 : 2) * cam::kGvWarps;
    const int64_t groups = (p->n_dim + columns - 1) / columns;
    // Offsets are data on the device: no more row blocks than rows.
    const int64_t grid = groups * p->rows, smem = static_cast<int64_t>(R) * p->k_dim * 2;
    if (grid > 0x7FFFFFFF || smem > cam::kGvMaxSmem) return static_cast<int>(cudaErrorInvalidValue);
    const cudaError_t err = limit.ensure(cam::expert_gemv_kernel<SWIGLU, FP16, R>, static_cast<int>(smem));
    if (err != cudaSuccess) return static_cast<int>(err);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1] = {cam::pdl_attribute()};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(cam::kGvThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, cam::expert_gemv_kernel<SWIGLU, FP16, R>, static_cast<const uint4*>(x), static_cast<const uint4*>(w), *p));
}

template <bool SWIGLU, bool FP16>
int launch_rows(const cam::GroupedMlpParams* p, const void* x, const void* w, cudaStream_t stream) {
    if (p->rows == 1) return launch_gemv<SWIGLU, FP16, 1>(p, x, w, stream);
    if (p->rows == 2) return launch_gemv<SWIGLU, FP16, 2>(p, x, w, stream);
    return launch_gemv<SWIGLU, FP16, 4>(p, x, w, stream);
}

}  // namespace

extern "C" int cam_launch_expert_gemv(const cam::GroupedMlpParams* p, int swiglu, const void* x, const void* w, cudaStream_t stream) {
    if (swiglu) return p->fp16 ? launch_rows<true, true>(p, x, w, stream) : launch_rows<true, false>(p, x, w, stream);
    return p->fp16 ? launch_rows<false, true>(p, x, w, stream) : launch_rows<false, false>(p, x, w, stream);
}
