// quantize_fp4 / dequantize_fp4: rows (or weights) to e2m1 codes with block scales and back; ../common/fp4.cuh has the format.
//
// A thread owns 16 consecutive values: one nvfp4 block, or half of an mxfp4 block whose maximum it exchanges with its
// neighbour.  Rows are whole blocks, so the tensor is one flat array of them and the scales come out in row order.
// Bound by memory: 2 bytes (bf16) in, 0.56 out per value.  32768 x 7168 bf16 to nvfp4 and back in a steady loop, 1.2 GB: 195 us
// (191 to 198 on several boards), 6.2 TB/s, 0.96 of a plain copy's rate.  Accesses of 32 bytes per thread fill whole sectors; with 16
// bytes the same took 242 us.
#include "../common/fp4.cuh"
#include "expert_ops.h"

namespace cam {

namespace {

constexpr int kQThreads = 256;
constexpr int kQPer = 2;  // groups of 16 values per thread, loads of all in flight together

// 32 bytes per thread at a time: a warp's accesses are whole sectors
__device__ __forceinline__ void load32(uint4* v, const uint4* p) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0].x), "=r"(v[0].y), "=r"(v[0].z), "=r"(v[0].w), "=r"(v[1].x), "=r"(v[1].y), "=r"(v[1].z), "=r"(v[1].w)
                 : "l"(p));
}
__device__ __forceinline__ void store32(uint4* p, const uint32_t* v) {
    asm volatile("st.global.L1::no_allocate.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

template <int DT>
struct Raw16;  // sixteen values as loaded
template <>
struct Raw16<0> { uint4 v[2]; };
template <>
struct Raw16<1> { uint4 v[2]; };
template <>
struct Raw16<2> { uint4 v[4]; };

template <int DT>
__device__ __forceinline__ void widen(const Raw16<DT>& r, float (&f)[16]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(r.v);
    if constexpr (DT == kDtFp32) {
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (DT == kDtBf16) {
                f[2 * i] = __uint_as_float(w[i] << 16);
                f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            } else {
                const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                f[2 * i] = t.x;
                f[2 * i + 1] = t.y;
            }
        }
    }
}

template <class Kernel, class... Args>
int launch_flat(Kernel kernel, int64_t groups, cudaStream_t stream, Args... args) {
    const int64_t per = kQThreads * kQPer, grid = (groups + per - 1) / per;
    if (grid > 0x7FFFFFFF) return static_cast<int>(cudaErrorInvalidValue);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1] = {pdl_attribute()};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(kQThreads);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, args...));
}

// 16-bit rows: six blocks per SM (40 registers), 32768 x 7168 bf16 to nvfp4 94 us; with the four that 52 registers leave 101.
template <int FMT, int DT>
__global__ void __launch_bounds__(kQThreads, DT == kDtFp32 ? 4 : 6)
quantize_fp4_kernel(const uint4* __restrict__ x, uint2* __restrict__ q, uint8_t* __restrict__ s, int64_t groups,
                    const float* __restrict__ gscale, int64_t groups_per_scale) {
    constexpr int V = DT == kDtFp32 ? 4 : 2;  // 16-byte loads of a group
    const int64_t base = static_cast<int64_t>(blockIdx.x) * (kQThreads * kQPer) + threadIdx.x;
    pdl_wait();
    pdl_release();
    Raw16<DT> r[kQPer];
#pragma unroll
    for (int u = 0; u < kQPer; ++u) {
        const int64_t i = base + u * kQThreads;
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            if (i < groups) load32(r[u].v + j, x + i * V + j);
            else r[u].v[j] = r[u].v[j + 1] = make_uint4(0, 0, 0, 0);
        }
    }
#pragma unroll
    for (int u = 0; u < kQPer; ++u) {
        const int64_t i = base + u * kQThreads;
        float f[16];
        widen<DT>(r[u], f);
        uint32_t amax = 0u;
#pragma unroll
        for (int j = 0; j < 16; ++j) amax = max(amax, __float_as_uint(f[j]) & 0x7FFFFFFFu);
        if (FMT == kFp4Mx) amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));  // blocks are pairs of lanes
        if (i >= groups) continue;
        float g = 1.f;
        if (FMT == kFp4Nv && gscale != nullptr) g = __ldg(gscale + (groups_per_scale > 0 ? i / groups_per_scale : 0));
        Fp4Divisor div;
        const uint32_t code = fp4_scale<FMT>(amax, g, __fmul_rn(6.f, g), div);
        q[i] = fp4_codes16<FMT>(f, div);
        if (FMT == kFp4Nv) s[i] = static_cast<uint8_t>(code);
        else if ((i & 1) == 0) s[i >> 1] = static_cast<uint8_t>(code);
    }
}

template <int FMT, int DT>
__global__ void __launch_bounds__(kQThreads)
dequantize_fp4_kernel(const uint2* __restrict__ q, const uint8_t* __restrict__ s, uint4* __restrict__ out, int64_t groups,
                      const float* __restrict__ gscale, int64_t groups_per_scale) {
    constexpr int V = DT == kDtFp32 ? 4 : 2;
    const int64_t base = static_cast<int64_t>(blockIdx.x) * (kQThreads * kQPer) + threadIdx.x;
    pdl_wait();
    pdl_release();
    uint2 c[kQPer];
    uint32_t sc[kQPer];
#pragma unroll
    for (int u = 0; u < kQPer; ++u) {
        const int64_t i = base + u * kQThreads;
        c[u] = i < groups ? __ldg(q + i) : make_uint2(0, 0);
        sc[u] = i < groups ? __ldg(s + (FMT == kFp4Nv ? i : i >> 1)) : 0u;
    }
#pragma unroll
    for (int u = 0; u < kQPer; ++u) {
        const int64_t i = base + u * kQThreads;
        if (i >= groups) continue;
        float d = FMT == kFp4Nv ? e4m3_value(sc[u]) : e8m0_value(sc[u]);
        if (FMT == kFp4Nv && gscale != nullptr) d = __fmul_rn(d, __ldg(gscale + (groups_per_scale > 0 ? i / groups_per_scale : 0)));
        uint32_t h[8];
        unpack_e2m1x8(c[u].x, *reinterpret_cast<uint32_t(*)[4]>(h));
        unpack_e2m1x8(c[u].y, *reinterpret_cast<uint32_t(*)[4]>(h + 4));
        uint32_t o[4 * V];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
            const float a = t.x * d, b = t.y * d;
            if constexpr (DT == kDtFp32) {
                o[2 * j] = __float_as_uint(a);
                o[2 * j + 1] = __float_as_uint(b);
            } else if constexpr (DT == kDtBf16) {
                const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
                o[j] = *reinterpret_cast<const uint32_t*>(&p);
            } else {
                const __half2 p = __floats2half2_rn(a, b);
                o[j] = *reinterpret_cast<const uint32_t*>(&p);
            }
        }
#pragma unroll
        for (int j = 0; j < V; j += 2) store32(out + i * V + j, o + 4 * j);
    }
}

}  // namespace

}  // namespace cam

// x: `groups` groups of 16 values; gscale: null, one float, or one per `groups_per_scale` groups (> 0).
extern "C" int cam_launch_quantize_fp4(const void* x, int dtype, int fmt, void* q, void* s, int64_t groups,
                                       const float* gscale, int64_t groups_per_scale, cudaStream_t stream) {
    using namespace cam;
    if (groups <= 0) return 0;
    auto go = [&](auto kernel) {
        return launch_flat(kernel, groups, stream, static_cast<const uint4*>(x), static_cast<uint2*>(q), static_cast<uint8_t*>(s), groups, gscale, groups_per_scale);
    };
    if (fmt == kFp4Nv)
        return dtype == kDtBf16 ? go(quantize_fp4_kernel<kFp4Nv, kDtBf16>) : dtype == kDtFp16 ? go(quantize_fp4_kernel<kFp4Nv, kDtFp16>) : go(quantize_fp4_kernel<kFp4Nv, kDtFp32>);
    return dtype == kDtBf16 ? go(quantize_fp4_kernel<kFp4Mx, kDtBf16>) : dtype == kDtFp16 ? go(quantize_fp4_kernel<kFp4Mx, kDtFp16>) : go(quantize_fp4_kernel<kFp4Mx, kDtFp32>);
}

extern "C" int cam_launch_dequantize_fp4(const void* q, const void* s, int dtype, int fmt, void* out, int64_t groups,
                                         const float* gscale, int64_t groups_per_scale, cudaStream_t stream) {
    using namespace cam;
    if (groups <= 0) return 0;
    auto go = [&](auto kernel) {
        return launch_flat(kernel, groups, stream, static_cast<const uint2*>(q), static_cast<const uint8_t*>(s), static_cast<uint4*>(out), groups, gscale, groups_per_scale);
    };
    if (fmt == kFp4Nv)
        return dtype == kDtBf16 ? go(dequantize_fp4_kernel<kFp4Nv, kDtBf16>) : dtype == kDtFp16 ? go(dequantize_fp4_kernel<kFp4Nv, kDtFp16>) : go(dequantize_fp4_kernel<kFp4Nv, kDtFp32>);
    return dtype == kDtBf16 ? go(dequantize_fp4_kernel<kFp4Mx, kDtBf16>) : dtype == kDtFp16 ? go(dequantize_fp4_kernel<kFp4Mx, kDtFp16>) : go(dequantize_fp4_kernel<kFp4Mx, kDtFp32>);
}
