// rms_norm / add_rms_norm, the same with rows in 8 bits, and their backward pass.
//
//   s = x + residual (rounded to the residual's type),  r = 1 / sqrt(mean(s^2) + eps),  y = s r w
//   dx = dresidual = ds + r (w dy - s r mean(w dy s r)),   dw = sum over the rows of dy s r
//
// Bound by memory in both directions, with the issue slots close behind: arithmetic runs on pairs (16-bit sums in one instruction,
// products and sums of two fp32 values in one).  16384 x 4096 with an fp32 residual 119 us, 32768 x 7168 to e4m3 or int8 240 us
// (1.03 of a plain copy's rate all), backward 8192 x 7168 bf16 81 us (0.88).  A row stays in the registers of the threads that share it: read once, summed, scaled and
// written.  A thread owns 16 consecutive values at a time, so blocks of 128 for e4m3 are eight lanes.  The norm is that of the
// rounded sum, so a backward pass (or a later layer) that reads the stored sum sees the numbers that were normalised.
#include "../common/quant.cuh"
#include "launch.h"
#include "layer_ops.h"
#include "layer_values.cuh"

namespace cam {

namespace {

// Rows alone, or the quant modes.  The two kinds of e4m3 scales are kernels of their own: in one kernel the divisions of the one spill registers of
// both, 32768 x 7168 bf16 with a residual 250 and 252 us instead of 238, without 167 and 170 instead of 156 and 159.
constexpr int kRowsOnly = 0, kInt8 = 2, kE4m3 = 3, kE4m3PowerOfTwo = 4;
constexpr int kWarpRows = 8;  // rows of a block where a row belongs to a warp

// ------------------------------------------------------------------------------------------------
// Sixteen values as they lie in memory
// ------------------------------------------------------------------------------------------------
template <int DT>
constexpr int kWords = DT == kDtFp32 ? 16 : 8;  // 32-bit words of sixteen values

template <int DT>
struct Raw16 {
    uint32_t w[kWords<DT>];
};

template <int DT>
__device__ __forceinline__ Pair widen2(const Raw16<DT>& r, int i) {
    if constexpr (DT == kDtFp32) return pair(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
    else if constexpr (DT == kDtBf16) return pair(__uint_as_float(r.w[i] << 16), __uint_as_float(r.w[i] & 0xFFFF0000u));
    else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
        return pair(f.x, f.y);
    }
}
template <int DT>
__device__ __forceinline__ void narrow2(Raw16<DT>& r, int i, Pair v) {
    const float2 f = split(v);
    if constexpr (DT == kDtFp32) {
        r.w[2 * i] = __float_as_uint(f.x);
        r.w[2 * i + 1] = __float_as_uint(f.y);
    } else if constexpr (DT == kDtBf16) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(f.x, f.y);
        r.w[i] = *reinterpret_cast<const uint32_t*>(&b);
    } else {
        const __half2 b = __floats2half2_rn(f.x, f.y);
        r.w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
}
// x + r of one type, rounded once
template <int DT>
__device__ __forceinline__ Raw16<DT> add16(const Raw16<DT>& x, const Raw16<DT>& r) {
    Raw16<DT> s;
#pragma unroll
    for (int i = 0; i < kWords<DT>; ++i) {
        if constexpr (DT == kDtFp32) s.w[i] = __float_as_uint(__uint_as_float(x.w[i]) + __uint_as_float(r.w[i]));
        else if constexpr (DT == kDtBf16) {
            const __nv_bfloat162 v = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&x.w[i]), *reinterpret_cast<const __nv_bfloat162*>(&r.w[i]));
            s.w[i] = *reinterpret_cast<const uint32_t*>(&v);
        } else {
            const __half2 v = __hadd2(*reinterpret_cast<const __half2*>(&x.w[i]), *reinterpret_cast<const __half2*>(&r.w[i]));
            s.w[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    return s;
}

// How rows can be read: 32 bytes at a time, 16 (rows of a multiple of 8 values), or one value (other widths, operands that are not
// aligned)
constexpr int kBy32 = 16, kBy16 = 8, kByOne = 1;

// Where a thread's values of a row lie
struct Place {
    int64_t row0;  // first value of the row
    int t, threads, h;
};

// Pairs of a piece: sixteen values, but eight where they go one by one, so that twice the threads have loads in flight: 8192 x 4095 bf16
// 88 us instead of 103, 20000 x 1023 fp16 50 instead of 63.
template <int VEC>
constexpr int kPairs = VEC == kByOne ? 4 : 8;

// Column of the first value of a thread's piece (kByOne: of value j)
template <int VEC>
__device__ __forceinline__ int column(const Place& at, int v, int j) {
    return VEC == kByOne ? (v * 8 + j) * at.threads + at.t : (v * at.threads + at.t) * 16 + j;
}

// Zeros past the row
template <int DT, int VEC>
__device__ __forceinline__ Raw16<DT> load16(const void* base, const Place& at, int v) {
    Raw16<DT> r;
    const int c = column<VEC>(at, v, 0);
    const char* p = static_cast<const char*>(base) + (at.row0 + c) * kBytes<DT>;
    if constexpr (VEC == kByOne) {
#pragma unroll
        for (int j = 0; j < 2 * kPairs<VEC>; ++j) {
            const int d = column<VEC>(at, v, j);
            if constexpr (DT == kDtFp32) r.w[j] = d < at.h ? __float_as_uint(load1<DT>(base, at.row0 + d)) : 0u;
            else {
                const uint32_t b = d < at.h ? __ldg(static_cast<const unsigned short*>(base) + at.row0 + d) : 0u;
                r.w[j / 2] = j % 2 ? r.w[j / 2] | b << 16 : b;
            }
        }
    } else if constexpr (VEC == kBy32) {
        if (c < at.h) {
            load32(r.w, p);
            if constexpr (DT == kDtFp32) {
                if (c + 8 < at.h) {
                    load32(r.w + 8, p + 32);
                } else {
#pragma unroll
                    for (int i = 8; i < 16; ++i) r.w[i] = 0u;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kWords<DT>; ++i) r.w[i] = 0u;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kWords<DT>; i += 4) {
            const int d = c + i * 4 / kBytes<DT>;
            uint4 q = make_uint4(0u, 0u, 0u, 0u);
            if (d < at.h) q = load16_stream(p + i * 4);
            r.w[i] = q.x, r.w[i + 1] = q.y, r.w[i + 2] = q.z, r.w[i + 3] = q.w;
        }
    }
    return r;
}

template <int DT, int VEC>
__device__ __forceinline__ void store16(void* base, const Place& at, int v, const Raw16<DT>& r) {
    const int c = column<VEC>(at, v, 0);
    char* p = static_cast<char*>(base) + (at.row0 + c) * kBytes<DT>;
    if constexpr (VEC == kByOne) {
#pragma unroll
        for (int j = 0; j < 2 * kPairs<VEC>; ++j) {
            const int d = column<VEC>(at, v, j);
            if (d >= at.h) continue;
            if constexpr (DT == kDtFp32) static_cast<uint32_t*>(base)[at.row0 + d] = r.w[j];
            else static_cast<unsigned short*>(base)[at.row0 + d] = static_cast<unsigned short>(r.w[j / 2] >> (j % 2 * 16));
        }
    } else if constexpr (VEC == kBy32) {
        if (c < at.h) {
            store32(p, r.w);
            if constexpr (DT == kDtFp32) {
                if (c + 8 < at.h) store32(p + 32, r.w + 8);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < kWords<DT>; i += 4) {
            const int d = c + i * 4 / kBytes<DT>;
            if (d < at.h) *reinterpret_cast<uint4*>(p + i * 4) = make_uint4(r.w[i], r.w[i + 1], r.w[i + 2], r.w[i + 3]);
        }
    }
}

// Weights of a thread's sixteen columns, which every row reads: through L1
template <int DT, int VEC>
__device__ __forceinline__ void load_weight_as(const void* w, const Place& at, int v, Pair* out) {
    Raw16<DT> r;
    if constexpr (VEC == kByOne) {
        Place first = at;
        first.row0 = 0;
        r = load16<DT, VEC>(w, first, v);
    } else {
        const int c = column<VEC>(at, v, 0);
        const char* p = static_cast<const char*>(w);
#pragma unroll
        for (int i = 0; i < kWords<DT>; i += 4) {
            const int d = c + i * 4 / kBytes<DT>;
            uint4 q = make_uint4(0u, 0u, 0u, 0u);
            if (d < at.h) q = __ldg(reinterpret_cast<const uint4*>(p + static_cast<int64_t>(d) * kBytes<DT>));
            r.w[i] = q.x, r.w[i + 1] = q.y, r.w[i + 2] = q.z, r.w[i + 3] = q.w;
        }
    }
#pragma unroll
    for (int i = 0; i < kPairs<VEC>; ++i) out[i] = widen2<DT>(r, i);
}
template <int DT, int VEC>
__device__ __forceinline__ void load_weight(const void* w, bool fp32, const Place& at, int v, Pair* out) {
    if (DT == kDtFp32 || fp32) load_weight_as<kDtFp32, VEC>(w, at, v, out);
    else load_weight_as<DT, VEC>(w, at, v, out);
}

// Sum (and maximum) over the threads that share a row, with one barrier: `red`, 64 floats of the block, is one of two that take turns
// where there are several rows.  The warps' sums are added in their order.
template <bool WARP, int N>
__device__ __forceinline__ void clear_sums(float (&red)[N]) {
    // places of warps that the block does not have; the first barrier comes before they are read
    if (!WARP && threadIdx.x < N && (threadIdx.x & 31) >= blockDim.x >> 5) red[threadIdx.x] = 0.f;
    if (!WARP && blockDim.x < N && threadIdx.x + blockDim.x < N && ((threadIdx.x + blockDim.x) & 31) >= blockDim.x >> 5) red[threadIdx.x + blockDim.x] = 0.f;
}
// Magnitudes compare as integers, and NaN is the largest.
__device__ __forceinline__ float larger(float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); }
__device__ __forceinline__ float widest(float top, float a, float b) {
    asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(a), "f"(b));
    return top;
}

template <bool WARP, bool MAX>
__device__ __forceinline__ void over_row(float& sum, float& top, float* red) {
    sum = warp_sum(sum);
    if (MAX) top = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top)));
    if constexpr (WARP) {
        __syncwarp();
    } else {
        const int warps = blockDim.x >> 5;
        if ((threadIdx.x & 31) == 0) {
            red[threadIdx.x >> 5] = sum;
            if (MAX) red[32 + (threadIdx.x >> 5)] = top;
        }
        __syncthreads();
        sum = 0.f;
#pragma unroll 4
        for (int i = 0; i < warps; i += 4) {  // what is behind the last warp is zero
            const float4 v = *reinterpret_cast<const float4*>(red + i);
            sum += v.x + v.y + (v.z + v.w);
            if (MAX) {
                const float4 m = *reinterpret_cast<const float4*>(red + 32 + i);
                top = larger(larger(top, larger(m.x, m.y)), larger(m.z, m.w));
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------
// Forward
// ------------------------------------------------------------------------------------------------
// Sixteen values of a row in 8 bits.  Adding 1.5 x 2^23 rounds to the nearest whole number and leaves it in the low byte; no value is above
// 127 / inv.  A conversion and a clamp for each took 257 us for 32768 x 7168 bf16
// instead of 235 (142 with the registers below).  inv is NaN for a row with NaN, or with an
// infinity before the norm, and zero for one with an infinity behind it: its scale says so, its values are zero.
template <int VEC>
__device__ __forceinline__ void store_int8(void* q, const Place& at, int v, const Pair* y, float inv) {
    const uint32_t keep = inv > 0.f ? 0xFFFFFFFFu : 0u;
    const Pair inv2 = pair(inv, inv), whole = pair(12582912.f, 12582912.f);
    uint32_t o[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < kPairs<VEC>; j += 2) {
        const float2 a = split(add2(mul2(y[j], inv2), whole)), b = split(add2(mul2(y[j + 1], inv2), whole));
        const uint32_t lo = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), hi = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
        o[j / 2] = __byte_perm(lo, hi, 0x5410) & keep;
    }
    int8_t* row = static_cast<int8_t*>(q) + at.row0;
#pragma unroll
    for (int i = 0; i < kPairs<VEC> / 4; ++i) {
        const int c = column<VEC>(at, v, VEC == kByOne ? 0 : 8 * i);
        if constexpr (VEC != kByOne) {
            if (c < at.h) *reinterpret_cast<uint2*>(row + c) = make_uint2(o[2 * i], o[2 * i + 1]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int d = column<VEC>(at, v, 8 * i + j);
                if (d < at.h) row[d] = static_cast<int8_t>(o[2 * i + j / 4] >> (j % 4 * 8));
            }
        }
    }
}

// Power-of-two scale: the least 2^k >= max(amax, 1e-4) / 448.  448 = 1.75 x 2^8, so k is the exponent of amax less 8, one more where the
// significand is above 1.75: exact, without a division.  A block with NaN has a NaN scale and NaN codes; one with an infinity has an
// infinite scale, NaN in the infinity's place and zeros in the others, so no product of it is finite.
__device__ __forceinline__ void block_scale(float amax, bool power_of_two, float& scale, float& inv) {
    const float a = larger(amax, 1e-4f);
    if (power_of_two) {
        const uint32_t b = __float_as_uint(a), e = (b >> 23) - 8u + ((b & 0x7FFFFFu) > 0x600000u ? 1u : 0u);
        const bool finite = b < 0x7F800000u;
        scale = finite ? __uint_as_float(e << 23) : a;
        inv = finite ? __uint_as_float((254u - e) << 23) : b == 0x7F800000u ? 0.f : a;
    } else {
        scale = a / 448.f;  // both divided as the dispatch does: the same bits from the same rows
        inv = 448.f / a;
    }
}

// Blocks of an SM, as a bound on registers.  Rows in 8 bits: 64 instead of 80 and 86, so that four blocks of 7168 columns have loads on their way
// and not three: 32768 x 7168 bf16 to e4m3 174 -> 144 us (150 to 158 with what marks blocks that are not finite), to int8 235 -> 142, with a residual
// 244 -> 239 and 294 -> 237; fp32 does not fit
// (16384 x 4096 with a residual to int8 128 -> 137).  Values one by one: 32 registers, 8192 x 4095 bf16 to int8 92 us, with 50 127.
template <int DT, int MODE, int NP, int VEC, bool WARP>
constexpr int kNormBlocks = !WARP && (VEC == kByOne ? NP == 1 : NP == 2 && MODE != kRowsOnly && DT != kDtFp32) ? 2 : 1;

template <int DT, int MODE, int NP, int VEC, bool WARP>
__global__ void __launch_bounds__(WARP ? kWarpRows * 32 : NP == 2 && VEC != kByOne ? 512 : 1024, kNormBlocks<DT, MODE, NP, VEC, WARP>)
rms_norm_kernel(const RmsNormParams p) {
    __shared__ __align__(16) float red[64];
    clear_sums<WARP>(red);
    const int threads = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x, h = p.h;
    const int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * kWarpRows + (threadIdx.x >> 5) : blockIdx.x, row0 = row * h;
    const Place at{row0, t, threads, h};
    pdl_wait();
    pdl_release();
    if (WARP && row >= p.rows) return;
    Pair s[NP][kPairs<VEC>];
    {
        Raw16<DT> x[NP];
#pragma unroll
        for (int v = 0; v < NP; ++v) x[v] = load16<DT, VEC>(p.x, at, v);
        if (p.residual == nullptr) {
#pragma unroll
            for (int v = 0; v < NP; ++v) {
#pragma unroll
                for (int i = 0; i < kPairs<VEC>; ++i) s[v][i] = widen2<DT>(x[v], i);
            }
        } else if (DT != kDtFp32 && p.res_type == kDtFp32) {
            Raw16<kDtFp32> r[NP];
#pragma unroll
            for (int v = 0; v < NP; ++v) r[v] = load16<kDtFp32, VEC>(p.residual, at, v);
#pragma unroll
            for (int v = 0; v < NP; ++v) {
#pragma unroll
                for (int i = 0; i < kPairs<VEC>; ++i) {
                    s[v][i] = add2(widen2<DT>(x[v], i), widen2<kDtFp32>(r[v], i));
                    narrow2<kDtFp32>(r[v], i, s[v][i]);
                }
                store16<kDtFp32, VEC>(p.sum, at, v, r[v]);
            }
        } else {
            Raw16<DT> r[NP];
#pragma unroll
            for (int v = 0; v < NP; ++v) r[v] = load16<DT, VEC>(p.residual, at, v);
#pragma unroll
            for (int v = 0; v < NP; ++v) {
                r[v] = add16<DT>(x[v], r[v]);
#pragma unroll
                for (int i = 0; i < kPairs<VEC>; ++i) s[v][i] = widen2<DT>(r[v], i);
                store16<DT, VEC>(p.sum, at, v, r[v]);
            }
        }
    }
    Pair squares = 0ull;
#pragma unroll
    for (int v = 0; v < NP; ++v) {
#pragma unroll
        for (int i = 0; i < kPairs<VEC>; ++i) squares = fma2(s[v][i], s[v][i], squares);
    }
    const float2 halves = split(squares);
    float sum = halves.x + halves.y, top = 0.f;
    // times the weight already: int8 needs the largest product along with the sum
#pragma unroll
    for (int v = 0; v < NP; ++v) {
        Pair w[kPairs<VEC>];
        load_weight<DT, VEC>(p.weight, p.weight_type == kDtFp32, at, v, w);
#pragma unroll
        for (int i = 0; i < kPairs<VEC>; ++i) {
            s[v][i] = mul2(s[v][i], w[i]);
            if (MODE == kInt8) {
                const float2 f = split(s[v][i]);
                top = widest(top, f.x, f.y);
            }
        }
    }
    over_row<WARP, MODE == kInt8>(sum, top, red);
    const float rstd = 1.f / sqrtf(sum / static_cast<float>(h) + p.eps);
    if (p.rstd != nullptr && t == 0) p.rstd[row] = rstd;
    const Pair rstd2 = pair(rstd, rstd);
    const float inv8 = 127.f / (top * rstd + 1e-12f);
    if (MODE == kInt8 && t == 0) p.scales[row] = 1.f / inv8;
#pragma unroll
    for (int v = 0; v < NP; ++v) {
#pragma unroll
        for (int i = 0; i < kPairs<VEC>; ++i) s[v][i] = mul2(s[v][i], rstd2);
        if (MODE == kRowsOnly || p.y != nullptr) {
            Raw16<DT> y;
#pragma unroll
            for (int i = 0; i < kPairs<VEC>; ++i) narrow2<DT>(y, i, s[v][i]);
            store16<DT, VEC>(p.y, at, v, y);
        }
        if constexpr (MODE == kInt8) store_int8<VEC>(p.q, at, v, s[v], inv8);
        if constexpr (MODE == kE4m3 || MODE == kE4m3PowerOfTwo) {
            // a block of 128 values: eight consecutive lanes
            float amax = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 f = split(s[v][i]);
                amax = widest(amax, f.x, f.y);
            }
#pragma unroll
            for (int o = 4; o >= 1; o >>= 1) amax = larger(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
            float scale, inv;
            block_scale(amax, MODE == kE4m3PowerOfTwo, scale, inv);
            const Pair inv2 = pair(inv, inv);
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 a = split(mul2(s[v][2 * i], inv2)), b = split(mul2(s[v][2 * i + 1], inv2));
                o[i] = pack_e4m3x4(a.x, a.y, b.x, b.y);
            }
            const int c = column<VEC>(at, v, 0);
            if (c < h) {
                *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.q) + row0 + c) = make_uint4(o[0], o[1], o[2], o[3]);
                if ((t & 7) == 0) p.scales[row * (h / 128) + (c >> 7)] = scale;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------
// Backward
// ------------------------------------------------------------------------------------------------
// Rows are shared out to the blocks in turn; a thread keeps the sums of its columns' weight gradients over all of its rows, and the
// block's go to `partial`, which a second kernel adds up in a fixed order.
//
// With STAGES > 0 every thread has a ring of its own pieces of the rows ahead in shared memory: it reads only what it (fp32: its warp)
// copied, so a wait for its own copies is all that the data needs, and the copies of a later row go out when it has read the place that
// they go to.  8192 x 7168 bf16 without the ring: 177 us.

// Everything goes in halves of eight values, and the ring is read again after the exchange rather than kept, so that 64 registers do and
// two blocks of 7168 columns share an SM.

// Column of value j of half `i`.  The halves are eight consecutive values each, and so are a warp's: 16 bytes per thread that were a
// half of 32 consecutive ones would fetch every sector twice (8192 x 7168 bf16: 138 us).
template <int VEC>
__device__ __forceinline__ int half_column(const Place& at, int i, int j) {
    return VEC == kByOne ? (i * 8 + j) * at.threads + at.t : (i * at.threads + at.t) * 8 + j;
}

// Eight values of a row as pairs
template <int DT, int VEC>
__device__ __forceinline__ void load_half(const void* base, const Place& at, int i, Pair* out) {
    if constexpr (VEC == kByOne) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = half_column<VEC>(at, i, 2 * j), e = half_column<VEC>(at, i, 2 * j + 1);
            out[j] = pair(d < at.h ? load1<DT>(base, at.row0 + d) : 0.f, e < at.h ? load1<DT>(base, at.row0 + e) : 0.f);
        }
    } else {
        const int c = half_column<VEC>(at, i, 0);
        Raw8<DT> r = {};
        if (c < at.h) {
            if constexpr (DT == kDtFp32) load32(reinterpret_cast<uint32_t*>(r.v), static_cast<const float*>(base) + at.row0 + c);
            else r = load8<DT>(base, at.row0 + c);
        }
        float f[8];
        widen8<DT>(r, f);
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = pair(f[2 * j], f[2 * j + 1]);
    }
}
template <int DT, int VEC>
__device__ __forceinline__ void store_half(void* base, const Place& at, int i, const Pair* v) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 e = split(v[j]);
        f[2 * j] = e.x;
        f[2 * j + 1] = e.y;
    }
    if constexpr (VEC == kByOne) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int d = half_column<VEC>(at, i, j);
            if (d < at.h) store1<DT>(base, at.row0 + d, f[j]);
        }
    } else {
        const int c = half_column<VEC>(at, i, 0);
        const Raw8<DT> r = narrow8<DT>(f);
        if (c < at.h) {
            if constexpr (DT == kDtFp32) store32(static_cast<float*>(base) + at.row0 + c, reinterpret_cast<const uint32_t*>(r.v));
            else store8<DT>(base, at.row0 + c, r);
        }
    }
}

template <int DT>
constexpr int kCopies = kBytes<DT> / 2;  // 16-byte copies of eight values

// A thread's sixteen values of an operand to the ring; returns where the next operand's begin (`ring`, for the whole block or warp).  Eight
// fp32 values are 32 bytes: there a warp's copies take turns by 16 bytes, so that each fetches whole sectors, and a thread reads
// what others of its warp copied.
template <int DT>
__device__ __forceinline__ uint32_t ring_copy(uint32_t ring, int threads, int t, int h, const void* base, int64_t row0) {
    const int lane = t & 31;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < kCopies<DT>; ++j) {
            const int unit = DT == kDtFp32 ? (t - lane) * 2 + j * 32 + lane : t, c = i * threads * 8 + unit * (8 / kCopies<DT>);
            if (c < h)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring + (i * kCopies<DT> * threads + unit) * 16), "l"(static_cast<const char*>(base) + (row0 + c) * kBytes<DT>) : "memory");
        }
    }
    return ring + 2 * kCopies<DT> * threads * 16;
}
template <int DT>
__device__ __forceinline__ void ring_half(uint32_t ring, int i, int threads, int t, Pair* out) {
    Raw8<DT> r;
#pragma unroll
    for (int j = 0; j < kCopies<DT>; ++j)
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.v[j].x), "=r"(r.v[j].y), "=r"(r.v[j].z), "=r"(r.v[j].w) : "r"(ring + ((i * threads + t) * kCopies<DT> + j) * 16) : "memory");
    float f[8];
    widen8<DT>(r, f);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = pair(f[2 * j], f[2 * j + 1]);
}

// Registers of a thread at most; the launcher counts with them
template <int ST, int HALVES, int STAGES>
constexpr int kBackwardRegisters = HALVES == 1 ? 64 : STAGES == 0 ? 128 : ST == kDtFp32 ? 96 : 64;

// HALVES: eights of values per thread
template <int DT, int ST, int WT, int VEC, int HALVES, bool WARP, int THREADS, int STAGES>
__global__ void __launch_bounds__(THREADS, THREADS > 512 ? 1 : 65536 / (THREADS * kBackwardRegisters<ST, HALVES, STAGES>))
rms_norm_backward_kernel(const RmsNormBackwardParams p, uint32_t stage_bytes) {
    extern __shared__ __align__(16) uint8_t dynamic[];  // WARP: per warp; the stages, and at the end the warps' sums
    __shared__ __align__(16) float red[128];
    clear_sums<WARP>(red);
    const int threads = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x, warp = threadIdx.x >> 5, h = p.h;
    const int64_t first = WARP ? static_cast<int64_t>(blockIdx.x) * kWarpRows + warp : blockIdx.x;
    const int64_t step = WARP ? static_cast<int64_t>(gridDim.x) * kWarpRows : gridDim.x;
    const uint32_t slots = smem_u32(dynamic) + (WARP ? warp * STAGES * stage_bytes : 0u);
    pdl_wait();
    pdl_release();
    auto copy = [&](int64_t row, int stage) {
        if (row < p.rows) {
            uint32_t next = ring_copy<DT>(slots + stage * stage_bytes, threads, t, h, p.dy, row * h);
            next = ring_copy<ST>(next, threads, t, h, p.sum, row * h);
            if (p.dsum != nullptr) ring_copy<ST>(next, threads, t, h, p.dsum, row * h);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if constexpr (STAGES > 0) {
        // places past the row, which no copy ever reaches, are read with the others
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if ((i * threads + t) * 8 < h) continue;
            for (int stage = 0; stage < STAGES; ++stage) {
                uint32_t at = slots + stage * stage_bytes;
                for (int operand = 0; operand < (p.dsum != nullptr ? 3 : 2); ++operand) {
                    const int copies = operand == 0 ? kCopies<DT> : kCopies<ST>;
                    for (int j = 0; j < copies; ++j)
                        asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(at + ((i * threads + t) * copies + j) * 16), "r"(0u) : "memory");
                    at += 2 * copies * threads * 16;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < STAGES; ++i) copy(first + i * step, i);
    }
    Raw16<WT> w;  // as it lies in memory: sixteen values in two halves
#pragma unroll
    for (int i = 0; i < HALVES; ++i) {
        Pair f[4];
        load_half<WT, VEC>(p.weight, Place{0, t, threads, h}, i, f);
#pragma unroll
        for (int j = 0; j < 4; ++j) narrow2<WT>(w, 4 * i + j, f[j]);
    }
    Pair acc[4 * HALVES];
#pragma unroll
    for (int i = 0; i < 4 * HALVES; ++i) acc[i] = 0ull;
    int stage = 0, turn = 0;
    for (int64_t row = first; row < p.rows; row += step) {
        const Place at{row * h, t, threads, h};
        const float rstd = __ldg(p.rstd + row);
        const Pair rstd2 = pair(rstd, rstd);
        const uint32_t at_dy = slots + stage * stage_bytes, at_s = at_dy + 2 * kCopies<DT> * threads * 16, at_ds = at_s + 2 * kCopies<ST> * threads * 16;
        Pair dy[4 * HALVES], s[4 * HALVES];
        if constexpr (STAGES > 0) {
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES > 0 ? STAGES - 1 : 0) : "memory");
            if (DT == kDtFp32 || ST == kDtFp32) __syncwarp();
        } else {
#pragma unroll
            for (int i = 0; i < HALVES; ++i) {
                load_half<DT, VEC>(p.dy, at, i, dy + 4 * i);
                load_half<ST, VEC>(p.sum, at, i, s + 4 * i);
            }
        }
        Pair products = 0ull;
#pragma unroll
        for (int i = 0; i < HALVES; ++i) {
            Pair* g = dy + 4 * i;
            Pair* hat = s + 4 * i;
            if constexpr (STAGES > 0) {
                ring_half<DT>(at_dy, i, threads, t, g);
                ring_half<ST>(at_s, i, threads, t, hat);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                hat[j] = mul2(hat[j], rstd2);
                acc[4 * i + j] = fma2(g[j], hat[j], acc[4 * i + j]);
                g[j] = mul2(g[j], widen2<WT>(w, 4 * i + j));
                products = fma2(g[j], hat[j], products);
            }
        }
        const float2 sides = split(products);
        float along = sides.x + sides.y, none = 0.f;
        over_row<WARP, false>(along, none, red + turn * 64);
        turn ^= 1;
        const float share = -along / static_cast<float>(h);
        const Pair share2 = pair(share, share);
#pragma unroll
        for (int i = 0; i < HALVES; ++i) {
            Pair* g = dy + 4 * i;
            Pair* hat = s + 4 * i;
            Pair d[4] = {0ull, 0ull, 0ull, 0ull};
            if constexpr (STAGES > 0) {
                ring_half<DT>(at_dy, i, threads, t, g);
                ring_half<ST>(at_s, i, threads, t, hat);
                if (p.dsum != nullptr) ring_half<ST>(at_ds, i, threads, t, d);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    hat[j] = mul2(hat[j], rstd2);
                    g[j] = mul2(g[j], widen2<WT>(w, 4 * i + j));
                }
            } else {
                if (p.dsum != nullptr) load_half<ST, VEC>(p.dsum, at, i, d);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j] = fma2(rstd2, fma2(share2, hat[j], g[j]), d[j]);
            if (p.dx != nullptr) store_half<DT, VEC>(p.dx, at, i, d);
            if (p.dres != nullptr) store_half<ST, VEC>(p.dres, at, i, d);
        }
        if constexpr (STAGES > 0) {
            if (DT == kDtFp32 || ST == kDtFp32) __syncwarp();
            copy(row + STAGES * step, stage);
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
    }
    if (p.partial == nullptr) return;
    float* mine = p.partial + static_cast<int64_t>(blockIdx.x) * h;
    const Place cols_at{0, t, threads, h};
    if constexpr (WARP) {
        // all rings have been read: the memory takes the warps' sums
        float* cols = reinterpret_cast<float*>(dynamic);
        if (STAGES > 0) asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8 * HALVES; ++j) {
            const int c = half_column<VEC>(cols_at, j / 8, j % 8);
            const float2 f = split(acc[j / 2]);
            if (c < h) cols[warp * h + c] = j % 2 ? f.y : f.x;
        }
        __syncthreads();
        for (int c = threadIdx.x; c < h; c += blockDim.x) {
            float a = 0.f;
#pragma unroll
            for (int r = 0; r < kWarpRows; ++r) a += cols[r * h + c];
            mine[c] = a;
        }
    } else {
#pragma unroll
        for (int i = 0; i < HALVES; ++i) store_half<kDtFp32, VEC>(mine, cols_at, i, acc + 4 * i);
    }
}

// dw[c] = sum over the parts: 32 columns and 32 shares of the parts per block
template <int DT>
__global__ void __launch_bounds__(1024) add_parts_kernel(const float* __restrict__ partial, int parts, int h, void* dw) {
    __shared__ float red[32][33];
    const int lane = threadIdx.x & 31, share = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    pdl_wait();
    pdl_release();
    float a = 0.f;
    if (c < h) {
#pragma unroll 8
        for (int i = share; i < parts; i += 32) a += __ldg(partial + static_cast<int64_t>(i) * h + c);
    }
    red[share][lane] = a;
    __syncthreads();
    // a warp per column: the shares in a tree
    const float sum = warp_sum(red[lane][share]);
    const int col = blockIdx.x * 32 + share;
    if (lane == 0 && col < h) store1<DT>(dw, col, sum);
}

// ------------------------------------------------------------------------------------------------
// Launches
// ------------------------------------------------------------------------------------------------
// Threads that share a row and sixteens of values per thread (pieces).  They follow from the width alone: a row's sums are added in the same
// order however many rows there are.
struct Shape {
    bool warp;
    int threads, pieces;
};

Shape shape_of(int h, int most) {
    const int pieces = (h + 15) / 16;
    if (pieces <= 32 * most) return {true, kWarpRows * 32, pieces <= 32 ? 1 : 2};
    return {false, ((pieces + most - 1) / most + 31) / 32 * 32, most};
}
// The same for values that go one by one, by eights
Shape shape_by_eights(int h) {
    const int pieces = (h + 7) / 8;
    if (pieces <= 32) return {true, kWarpRows * 32, 1};
    return pieces <= 1024 ? Shape{false, (pieces + 31) / 32 * 32, 1} : Shape{false, ((pieces + 1) / 2 + 31) / 32 * 32, 2};
}
static_assert(kWarpRows * 32 == 256 && 512 * 2 * 16 >= kNormMaxHidden, "every row has its threads");

int64_t turns_of(const Shape& s, int64_t rows) { return s.warp ? (rows + kWarpRows - 1) / kWarpRows : rows; }

template <int DT, int MODE, int VEC>
int launch_norm(const RmsNormParams& p, cudaStream_t stream) {
    const Shape s = VEC == kByOne ? shape_by_eights(p.h) : shape_of(p.h, 2);
    const dim3 grid(static_cast<unsigned>(turns_of(s, p.rows)));
    // by eights a warp has one piece and a block one or two, by sixteens a warp has one or two and a block two
    constexpr int most = VEC == kByOne ? 1 : 2;
    if (s.warp) return s.pieces == 1 ? launch_pdl(rms_norm_kernel<DT, MODE, 1, VEC, true>, grid, s.threads, 0, stream, p) : launch_pdl(rms_norm_kernel<DT, MODE, most, VEC, true>, grid, s.threads, 0, stream, p);
    return s.pieces == 1 ? launch_pdl(rms_norm_kernel<DT, MODE, most, VEC, false>, grid, s.threads, 0, stream, p) : launch_pdl(rms_norm_kernel<DT, MODE, 2, VEC, false>, grid, s.threads, 0, stream, p);
}

// How all operands of a launch can be read.  32 bytes are sixteen values, or eight of a row of fp32: 23315 x 6328 fp32 378 us, 16 bytes at
// a time 525.
template <int DT, class... Pointers>
int access_of(int h, Pointers... ps) {
    if (h % (DT == kDtFp32 ? 8 : 16) == 0 && (aligned32(ps) && ...)) return kBy32;
    return h % 8 == 0 && (aligned16(ps) && ...) ? kBy16 : kByOne;
}

template <int DT>
int launch_norm_type(const RmsNormParams& p, cudaStream_t stream) {
    const int access = access_of<DT>(p.h, p.x, p.residual, p.weight, p.y, p.sum, p.q);
    if (p.quant_mode == 0)
        return access == kBy32 ? launch_norm<DT, kRowsOnly, kBy32>(p, stream) : access == kBy16 ? launch_norm<DT, kRowsOnly, kBy16>(p, stream) : launch_norm<DT, kRowsOnly, kByOne>(p, stream);
    if (p.quant_mode == 2)
        return access == kBy32 ? launch_norm<DT, kInt8, kBy32>(p, stream) : access == kBy16 ? launch_norm<DT, kInt8, kBy16>(p, stream) : launch_norm<DT, kInt8, kByOne>(p, stream);
    if (access == kByOne || p.h % 128 != 0) return static_cast<int>(cudaErrorInvalidValue);
    if (p.quant_mode == 4) return access == kBy32 ? launch_norm<DT, kE4m3PowerOfTwo, kBy32>(p, stream) : launch_norm<DT, kE4m3PowerOfTwo, kBy16>(p, stream);
    return access == kBy32 ? launch_norm<DT, kE4m3, kBy32>(p, stream) : launch_norm<DT, kE4m3, kBy16>(p, stream);
}

// A launch of the backward pass
struct Backward {
    Shape shape;
    int blocks;                     // of an SM
    int stages, stage_bytes, smem;  // stages: 0 without a ring
};

int blocks_by_registers(const Shape& s, int registers) { return s.threads > 512 ? 1 : 65536 / (registers * s.threads); }

// Values loaded one by one: eight per thread where a block has the threads for it.  8192 x 4095 bf16 107 us, with sixteen 197 us
// (128 registers a thread leave half the loads in flight).
int halves_of(int h, bool single) { return single && h <= 8192 ? 1 : 2; }

Backward backward_of(const RmsNormBackwardParams& p, int dtype, bool ring) {
    const int halves = halves_of(p.h, !ring);
    Backward r{halves == 1 ? shape_by_eights(p.h) : shape_of(p.h, 1), 0, 0, 0, 0};
    const int group = r.shape.warp ? 32 : r.shape.threads, groups = r.shape.threads / group;
    const int size = dtype == kDtFp32 ? 4 : 2, sum = p.sum_type == kDtFp32 ? 4 : size, copies = size + sum + (p.dsum != nullptr ? sum : 0);
    const int sums = r.shape.warp ? kWarpRows * p.h * 4 : 0, room = 220 * 1024;
    const Backward plain{r.shape, blocks_by_registers(r.shape, halves == 1 ? 64 : 128), 0, 0, sums};
    r.blocks = blocks_by_registers(r.shape, sum == 2 ? 64 : 96);
    // below two turns of all blocks there is nothing to load ahead
    if (!ring || turns_of(r.shape, p.rows) <= 2 * static_cast<int64_t>(r.blocks) * sm_count_of_current_device()) return plain;
    r.stage_bytes = group * 16 * copies;
    const int per_stage = r.stage_bytes * groups;
    // all blocks with four stages, or as many as fit with two
    r.stages = r.blocks * (4 * per_stage + 1024) <= room ? 4 : 2;
    r.smem = r.stages * per_stage > sums ? r.stages * per_stage : sums;
    const int fit = room / (r.smem + 1024);
    if (fit < 1) return plain;
    r.blocks = r.blocks < fit ? r.blocks : fit;
    return r;
}

template <int DT, int ST, int WT, int VEC, int HALVES, bool WARP, int THREADS, int STAGES>
int launch_backward_kernel(const RmsNormBackwardParams& p, const Backward& r, cudaStream_t stream) {
    static SmemLimitCache limit;
    auto kernel = rms_norm_backward_kernel<DT, ST, WT, VEC, HALVES, WARP, THREADS, STAGES>;
    const cudaError_t err = limit.ensure(kernel, r.smem);
    if (err != cudaSuccess) return static_cast<int>(err);
    return launch_pdl(kernel, dim3(static_cast<unsigned>(p.parts)), r.shape.threads, static_cast<size_t>(r.smem), stream, p, static_cast<uint32_t>(r.stage_bytes));
}

template <int DT, int ST, int WT, int VEC, int HALVES, int STAGES>
int launch_backward(const RmsNormBackwardParams& p, const Backward& r, cudaStream_t stream) {
    if (r.shape.warp) return launch_backward_kernel<DT, ST, WT, VEC, HALVES, true, 256, STAGES>(p, r, stream);
    return r.shape.threads <= 512 ? launch_backward_kernel<DT, ST, WT, VEC, HALVES, false, 512, STAGES>(p, r, stream) : launch_backward_kernel<DT, ST, WT, VEC, HALVES, false, 1024, STAGES>(p, r, stream);
}

template <int DT, int ST, int WT>
int launch_backward_types(RmsNormBackwardParams p, cudaStream_t stream) {
    int access = access_of<DT>(p.h, p.dy, p.dsum, p.sum, p.weight, p.dx, p.dres, p.partial);
    // fp32 goes by 32 bytes
    auto whole = [](int type, auto... ps) { return type != kDtFp32 || (aligned32(ps) && ...); };
    if (!whole(DT, p.dy, p.dx) || !whole(ST, p.sum, p.dsum, p.dres) || !whole(WT, p.weight) || !whole(kDtFp32, p.partial)) access = kByOne;
    const Backward r = backward_of(p, DT, access != kByOne);
    const int64_t blocks = static_cast<int64_t>(r.blocks) * sm_count_of_current_device();
    p.parts = static_cast<int>(p.parts < blocks ? p.parts : blocks);
    int rc;
    if (access == kByOne) rc = halves_of(p.h, true) == 1 ? launch_backward<DT, ST, WT, kByOne, 1, 0>(p, r, stream) : launch_backward<DT, ST, WT, kByOne, 2, 0>(p, r, stream);
    else rc = r.stages == 4 ? launch_backward<DT, ST, WT, kBy16, 2, 4>(p, r, stream) : r.stages == 2 ? launch_backward<DT, ST, WT, kBy16, 2, 2>(p, r, stream) : launch_backward<DT, ST, WT, kBy16, 2, 0>(p, r, stream);
    if (rc != 0 || p.dweight == nullptr) return rc;
    return launch_pdl(add_parts_kernel<WT>, dim3(static_cast<unsigned>((p.h + 31) / 32)), 1024, 0, stream, static_cast<const float*>(p.partial), p.parts, p.h, p.dweight);
}

template <int DT>
int launch_backward_type(const RmsNormBackwardParams& p, cudaStream_t stream) {
    if (DT == kDtFp32) return launch_backward_types<kDtFp32, kDtFp32, kDtFp32>(p, stream);
    if (p.sum_type == kDtFp32)
        return p.weight_type == kDtFp32 ? launch_backward_types<DT, kDtFp32, kDtFp32>(p, stream) : launch_backward_types<DT, kDtFp32, DT>(p, stream);
    return p.weight_type == kDtFp32 ? launch_backward_types<DT, DT, kDtFp32>(p, stream) : launch_backward_types<DT, DT, DT>(p, stream);
}

}  // namespace

}  // namespace cam

extern "C" int cam_launch_rms_norm(const cam::RmsNormParams* p, int dtype, cudaStream_t stream) {
    using namespace cam;
    return dtype == kDtBf16 ? launch_norm_type<kDtBf16>(*p, stream) : dtype == kDtFp16 ? launch_norm_type<kDtFp16>(*p, stream) : launch_norm_type<kDtFp32>(*p, stream);
}

// Most blocks that a launch for these rows has
extern "C" int cam_rms_norm_backward_blocks(int64_t rows, int h) {
    using namespace cam;
    // an upper bound: operands of a width in eights that are not aligned get by with what their aligned kin have
    const Shape s = h % 8 != 0 && halves_of(h, true) == 1 ? shape_by_eights(h) : shape_of(h, 1);
    const int64_t turns = turns_of(s, rows), most = static_cast<int64_t>(sm_count_of_current_device()) * blocks_by_registers(s, 64);
    return static_cast<int>(turns < most ? turns : most);
}

extern "C" int cam_launch_rms_norm_backward(const cam::RmsNormBackwardParams* p, int dtype, cudaStream_t stream) {
    using namespace cam;
    return dtype == kDtBf16 ? launch_backward_type<kDtBf16>(*p, stream) : dtype == kDtFp16 ? launch_backward_type<kDtFp16>(*p, stream) : launch_backward_type<kDtFp32>(*p, stream);
}
