// 4-bit floating point with block scales.
//   e2m1     values 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives; two to a byte, the even element in the low nibble
//   nvfp4    blocks of 16: s = e4m3(amax / (6 g)), q = e2m1(x / (s g)), x ~ q s g with one fp32 scale g per tensor or expert
//   mxfp4    blocks of 32: s = 2^k, the smallest with 2^k >= amax / 6 (k >= -126; an all-zero block has 2^-127), x ~ q s
// All roundings are to nearest, ties to even; what rounds to zero keeps its sign.  A NaN anywhere in an nvfp4 block makes its scale NaN (and with it the whole
// block); an infinity takes the largest scale and saturates to 6.  In mxfp4 NaN gives the scale code 255 (NaN), an
// infinity the scale 2^127.
#pragma once
#include "ptx.cuh"

namespace cam {

constexpr int kFp4Nv = 0, kFp4Mx = 1;  // formats
__host__ __device__ constexpr int fp4_block(int fmt) { return fmt == kFp4Nv ? 16 : 32; }

// Eight floats (already divided by their scale) to four bytes of e2m1, saturating.
__device__ __forceinline__ uint32_t pack_e2m1x8(float a0, float a1, float a2, float a3, float a4, float a5, float a6, float a7) {
    uint32_t r;
    asm("{\n"
        ".reg .b8 b0, b1, b2, b3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"  // the first source lands in the upper nibble
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
        "mov.b32 %0, {b0, b1, b2, b3};\n"
        "}\n"
        : "=r"(r)
        : "f"(a0), "f"(a1), "f"(a2), "f"(a3), "f"(a4), "f"(a5), "f"(a6), "f"(a7));
    return r;
}

// Four bytes of e2m1 to eight halves (every e2m1 value is exact in fp16).
__device__ __forceinline__ void unpack_e2m1x8(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n"
        ".reg .b8 b0, b1, b2, b3;\n"
        "mov.b32 {b0, b1, b2, b3}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n"
        "}\n"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}

__device__ __forceinline__ uint32_t e4m3_code(float v) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(v));
    return r & 0xFFu;
}
__device__ __forceinline__ float e4m3_value(uint32_t code) {
    __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(code), __NV_E4M3);
    return __half2float(*reinterpret_cast<__half*>(&h));
}
__device__ __forceinline__ float e8m0_value(uint32_t code) {  // 2^(code - 127); code 255 is NaN
    return __uint_as_float(code == 0u ? 0x00400000u : code == 255u ? 0x7FC00000u : code << 23);
}

// What the values of a block are divided by: d, and 1 / d rounded to nearest.
// nvfp4: a block is `plain` where the division can neither overflow nor lose bits below the range of fp32: with a global scale of 2^-50
// to 2^100 d is between 2^-59 and 2^109 (or 0, with all values below half of the smallest scale), and values below 2^64 have
// quotients below 2^123 (above 9 only where the block scale was cut to 448; they saturate).
struct Fp4Divisor {
    float d, inv;
    bool plain;
};

// The scale of a block from the bits of its largest magnitude: its code and the divisor.
// (The maximum of magnitudes as unsigned integers is the maximum of the values, with NaN above infinity.)
template <int FMT>
__device__ __forceinline__ uint32_t fp4_scale(uint32_t amax_bits, float g, float six_g, Fp4Divisor& q) {
    const float amax = __uint_as_float(amax_bits);
    if (FMT == kFp4Nv) {
        const uint32_t code = e4m3_code(__fdiv_rn(amax, six_g));
        q.d = __fmul_rn(e4m3_value(code), g);
        q.inv = q.d > 0.f ? __fdiv_rn(1.f, q.d) : 0.f;  // d is NaN for a NaN block, whose codes mean nothing
        q.plain = amax < 0x1p64f && g >= 0x1p-50f && g <= 0x1p100f;
        return code;
    }
    q.plain = true;
    if (amax_bits > 0x7F800000u) {
        q.d = amax;
        q.inv = 0.f;
        return 255u;
    }
    const uint32_t b = __float_as_uint(__fdiv_rn(amax, 6.f));
    uint32_t e = (b >> 23) + ((b & 0x7FFFFFu) ? 1u : 0u);
    e = e > 254u ? 254u : e;
    q.d = e8m0_value(e);
    q.inv = e == 254u ? __uint_as_float(0x00400000u) : e == 0u ? 0.f : __uint_as_float((254u - e) << 23);
    return e;
}

// Two floats at a time
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// -x / d rounded to nearest, for nvfp4: with t = x inv and inv = 1 / d rounded to nearest, one remainder step t + (x - t d) inv gives
// the correctly rounded quotient (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990),
// so that a quotient half-way between two e2m1 values is seen as one.  All of it is negated, because a remainder of zero is +0: added
// to t it would lose the sign of x = -0, subtracted from -t it does not.  In pairs the arithmetic of 32768 x 7168 bf16 values stays
// hidden behind memory (94 us; one at a time 99).
__device__ __forceinline__ void fp4_minus_quotients(const float* v, const Fp4Divisor& q, float (&y)[16]) {
    const uint64_t minus_inv = pair_of(-q.inv, -q.inv), d = pair_of(q.d, q.d);
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        const uint64_t x = pair_of(v[i], v[i + 1]), t = mul_pair(x, minus_inv), z = fma_pair(fma_pair(t, d, x), minus_inv, t);
        asm("mov.b64 {%0, %1}, %2;" : "=f"(y[i]), "=f"(y[i + 1]) : "l"(z));
    }
}
// The same for blocks that are not plain.  Below 2^-60 values and divisor are taken times 2^64: 1 / d overflows below 2^-128, and the
// remainder, 2^-48 of the value, is cut below 2^-101.  t is cut to 16, so that no remainder is infinity minus infinity; what is cut
// saturates whatever the step adds.  Beside an infinite d all values are nothing.
__device__ __forceinline__ void fp4_minus_quotients_any(const float* v, float d, float (&y)[16]) {
    const float lift = d > 0.f && d < 0x1p-60f ? 0x1p64f : 1.f;
    d = __float_as_uint(d) == 0x7F800000u ? 0.f : d * lift;
    const float inv = d > 0.f ? __fdiv_rn(1.f, d) : 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float x = v[i] * lift, t = fminf(fmaxf(x * inv, -16.f), 16.f);
        y[i] = copysignf(__fmaf_rn(__fmaf_rn(-t, d, x), inv, t), -x);
    }
}

// Sixteen floats, divided by d and rounded, to eight bytes of codes.  mxfp4 divides by a power of two: the product is exact.
template <int FMT>
__device__ __forceinline__ uint2 fp4_codes16(const float* v, const Fp4Divisor& q) {
    float y[16];
    if (FMT == kFp4Mx) {
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = v[i] * q.inv;
    } else if (q.plain) {
        fp4_minus_quotients(v, q, y);
    } else {
        fp4_minus_quotients_any(v, q.d, y);
    }
    const uint32_t flip = FMT == kFp4Mx ? 0u : 0x88888888u;  // the signs
    return make_uint2(pack_e2m1x8(y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]) ^ flip,
                      pack_e2m1x8(y[8], y[9], y[10], y[11], y[12], y[13], y[14], y[15]) ^ flip);
}

}  // namespace cam
