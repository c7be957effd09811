// Loads, stores and sums shared by the operators round the experts.  Rows are bf16, fp16 or fp32; arithmetic is fp32.
#pragma once
#include <cuda_fp16.h>

#include "../common/ptx.cuh"
#include "expert_ops.h"

namespace cam {

template <int DT>
constexpr int kBytes = DT == kDtFp32 ? 4 : 2;

// Pairs of fp32 values: one instruction for both
using Pair = unsigned long long;

__device__ __forceinline__ Pair pair(float a, float b) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 split(Pair v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// 32 bytes per thread at a time: whole sectors
__device__ __forceinline__ void load32(uint32_t* v, const void* p) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "l"(p));
}
__device__ __forceinline__ void store32(void* p, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

// eight consecutive values as they lie in memory
template <int DT>
struct Raw8 {
    uint4 v[DT == kDtFp32 ? 2 : 1];
};

__device__ __forceinline__ uint4 load16_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

template <int DT>
__device__ __forceinline__ Raw8<DT> load8(const void* base, int64_t i) {
    Raw8<DT> r;
    const char* p = static_cast<const char*>(base) + i * kBytes<DT>;
    r.v[0] = load16_stream(p);
    if constexpr (DT == kDtFp32) r.v[1] = load16_stream(p + 16);
    return r;
}

template <int DT>
__device__ __forceinline__ void widen8(const Raw8<DT>& r, float* f) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(r.v);
    if constexpr (DT == kDtFp32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
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

template <int DT>
__device__ __forceinline__ Raw8<DT> narrow8(const float* f) {
    Raw8<DT> r;
    uint32_t* w = reinterpret_cast<uint32_t*>(r.v);
    if constexpr (DT == kDtFp32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == kDtBf16) {
                const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&p);
            } else {
                const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&p);
            }
        }
    }
    return r;
}

template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t i, const Raw8<DT>& r) {
    uint4* p = reinterpret_cast<uint4*>(static_cast<char*>(base) + i * kBytes<DT>);
    p[0] = r.v[0];
    if constexpr (DT == kDtFp32) p[1] = r.v[1];
}

template <int DT>
__device__ __forceinline__ float load1(const void* base, int64_t i) {
    if constexpr (DT == kDtFp32) return __ldg(static_cast<const float*>(base) + i);
    const unsigned short b = __ldg(static_cast<const unsigned short*>(base) + i);
    if constexpr (DT == kDtBf16) return __uint_as_float(static_cast<uint32_t>(b) << 16);
    return __half2float(__ushort_as_half(b));
}

template <int DT>
__device__ __forceinline__ void store1(void* base, int64_t i, float v) {
    if constexpr (DT == kDtFp32) static_cast<float*>(base)[i] = v;
    else if constexpr (DT == kDtBf16) static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(base)[i] = __float2half_rn(v);
}

// ------------------------------------------------------------------------------------------------
// Rows of odd widths: 16 bytes from and to any address
// ------------------------------------------------------------------------------------------------
// Byte by byte: at the ends of the memory alone
static __device__ __noinline__ uint4 load_window_at_end(const char* at, const char* lo, const char* hi) {
    uint32_t r[4] = {0u, 0u, 0u, 0u};
    for (int i = 0; i < 16; ++i) {
        const uint32_t b = at + i >= lo && at + i < hi ? __ldg(reinterpret_cast<const unsigned char*>(at) + i) : 0u;
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] |= i / 4 == k ? b << (i % 4 * 8) : 0u;
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// Sixteen bytes from any address, of memory that reaches from lo to hi; what is outside comes as zeros.  Two aligned pieces, of which the
// second is the first one of a neighbouring thread and lies in L1, shifted together.
__device__ __forceinline__ uint4 load_window(const char* at, const char* lo, const char* hi) {
    const uint32_t d = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(at) & 15u);
    const char* a = at - d;
    if (a < lo || a + (d != 0u ? 32 : 16) > hi) return load_window_at_end(at, lo, hi);
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(a));
    if (d == 0u) return u;
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(a) + 1);
    uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
    if (d & 8u) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (d & 4u) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    const uint32_t bits = (d & 3u) * 8u;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// Elements of ES bytes at places from..to - 1 of a piece, which starts at an aligned address
template <int ES>
__device__ __forceinline__ void store_some(char* at, const uint4& v, int from, int to) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 16 / ES; ++i) {
        if (i < from || i >= to) continue;
        if constexpr (ES == 4) *reinterpret_cast<uint32_t*>(at + 4 * i) = w[i];
        else if constexpr (ES == 2) *reinterpret_cast<uint16_t*>(at + 2 * i) = static_cast<uint16_t>(w[i / 2] >> (i % 2 * 16));
        else *reinterpret_cast<uint8_t*>(at + i) = static_cast<uint8_t>(w[i / 4] >> (i % 4 * 8));
    }
}
// Zeros at the other places
template <int ES>
__device__ __forceinline__ uint4 keep_some(const uint4& v, int from, int to) {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 16 / ES; ++i) {
        if (i >= from && i < to) continue;
        if constexpr (ES == 4) w[i] = 0u;
        else w[i / 2] &= i % 2 ? 0x0000FFFFu : 0xFFFF0000u;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}

// A kernel launch that may start while its predecessor ends (programmatic dependent launch)
template <class Kernel, class... Args>
int launch_pdl(Kernel kernel, dim3 grid, int threads, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1] = {pdl_attribute()};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, args...));
}

__host__ __device__ inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
__host__ __device__ inline bool aligned32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; }

}  // namespace cam
