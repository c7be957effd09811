// What the grouped products of the stand-alone expert-MLP operators share: the walker over the tiles of ragged experts, the
// zero fill of rows that belong to no expert, the epilogue's staging of 16-bit rows and the launch on CTA pairs.
#pragma once
#include "../common/fp4.cuh"
#include "expert_ops.h"
#include "gemm_common.cuh"

namespace cam {

// ----------------------------------------------------------------------------------------
// Waits of the single-lane roles (TMA producer, MMA issuer).  The whole warp walks the loop and one elected lane issues, so
// that descriptors and counters stay uniform.  A look at an mbarrier takes about 130 cycles even when the phase is complete,
// a quarter of a K-block: the roles therefore look at the next stage's barrier before they issue the present one's work
// (mbar_test), and come back to it only if it was not complete then (mbar_wait_warp).
// ----------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok;
}
// A wait that ran out.  `st` lies in host memory that the device can write, where the next call, and the host at any time, sees it
// without a copy: one 16-byte store, unless an earlier one is there already.
__device__ __forceinline__ void record_status(CamStatus* st, int code, int who, int detail) {
    if (*reinterpret_cast<volatile int32_t*>(&st->code) != 0) return;
    asm volatile("st.volatile.global.v4.s32 [%0], {%1, %2, %3, %4};" ::"l"(st), "r"(code), "r"(who), "r"(detail), "r"(static_cast<int>(blockIdx.x)) : "memory");
    __threadfence_system();
}
// Bounded: after kWaitPolls polls (each of which the hardware may itself hold for a while), or once another role has given up,
// it returns with *abort set; the pipeline then runs to the end of its tile without waiting, its results mean nothing, and the CTA
// lets the copies in flight land (abort_drain) before it leaves.
constexpr uint32_t kWaitPolls = 1u << 23;
__device__ __forceinline__ void mbar_wait_warp(uint32_t bar, uint32_t parity, uint32_t abort) {
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        ".reg .b32 n, f;\n"
        "mov.u32 n, 0;\n"
        "POLL:\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%0], %1;\n"
        "@p bra DONE;\n"
        "add.u32 n, n, 1;\n"
        "and.b32 f, n, 255;\n"
        "setp.ne.u32 q, f, 0;\n"
        "@q bra POLL;\n"
        "ld.volatile.shared.u32 f, [%2];\n"
        "setp.ne.u32 q, f, 0;\n"
        "@q bra DONE;\n"
        "setp.lt.u32 q, n, %3;\n"
        "@q bra POLL;\n"
        "st.volatile.shared.u32 [%2], 1;\n"
        "DONE:\n"
        "}\n" ::"r"(bar), "r"(parity), "r"(abort), "n"(kWaitPolls)
        : "memory");
}
// Arrive on the barrier at this shared-memory offset in BOTH CTAs of the pair once every MMA issued so far by this thread has
// completed: one instruction instead of two.
__device__ __forceinline__ void tc_commit_both(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"(static_cast<uint16_t>(3))
                 : "memory");
}
// The same answer in all lanes of a converged warp
__device__ __forceinline__ bool aborted(const volatile uint32_t* abort_flag) { return __any_sync(0xFFFFFFFFu, *abort_flag != 0u); }
// After a wait that ran out copies may still be on their way to this CTA's shared memory: two milliseconds, where they take
// microseconds, before the memory is given up.
__device__ __forceinline__ void abort_drain(const volatile uint32_t* abort_flag) {
    if (*abort_flag == 0u) return;
    const uint64_t t0 = globaltimer_ns();
    for (int i = 0; i < 4000 && globaltimer_ns() - t0 < 2000000ull; ++i) __nanosleep(1000);
}
// The epilogue's wait for a tile.  The warps of an epilogue meet at named barriers, and a wait that runs out is not seen by all of them
// in the same tile: whoever left the tile loop alone would leave the others at a barrier for good.  So nobody leaves it.  After a wait
// that ran out a warp goes through the tiles that are left without waiting; what it writes means nothing (the status says so), every
// barrier has its threads and the loop ends.
__device__ __forceinline__ void epilogue_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag, uint32_t sleep_ns) {
    if (!mbar_try_wait(bar, parity) && *abort_flag == 0u) mbar_wait_bounded(bar, parity, abort_flag, 2000000000ull, sleep_ns);
    __syncwarp();
}
// Position in a ring of stages: stage and the parity of its current turn
struct Ring {
    uint32_t s = 0, ph = 0;
    __device__ __forceinline__ void next(uint32_t n) {
        if (++s == n) { s = 0; ph ^= 1u; }
    }
};

// Offsets are data on the device: whatever they hold, first and last row of an expert stay inside [0, rows].
__device__ __forceinline__ int expert_bound(const int* off, int i, int rows) { return min(max(__ldg(off + i), 0), rows); }

// Tiles of TM rows x n_tiles columns of every expert, expert by expert; the columns of a row block are neighbours.
template <int TM>
struct RowWalker {
    const int* off;
    int num_experts, n_tiles, rows_total;
    int e = 0, base = 0;
    __device__ RowWalker(const int* o, int ne, int nt, int rt) : off(o), num_experts(ne), n_tiles(nt), rows_total(rt) {}
    __device__ bool locate(int tile, int& e_out, int& nt, int& row0, int& rows) {
        while (e < num_experts) {
            const int first = expert_bound(off, e, rows_total);
            const int cnt = max(expert_bound(off, e + 1, rows_total) - first, 0);
            const int tiles = ((cnt + TM - 1) / TM) * n_tiles;
            if (tile < base + tiles) {
                const int local = tile - base, mt = local / n_tiles;
                nt = local - mt * n_tiles;
                row0 = first + mt * TM;
                rows = min(TM, cnt - mt * TM);
                e_out = e;
                return true;
            }
            base += tiles;
            ++e;
        }
        return false;
    }
};

using PairTileWalker = RowWalker<2 * BM>;

// Rows before the first and past the last expert get zeros (16-byte units, `pitch16` of them per row); called by `threads`
// threads of every CTA, `t` their index.
__device__ __forceinline__ void zero_loose_rows(void* out, int64_t pitch16, const int* off, int num_experts, int rows, int t, int threads) {
    const int head = expert_bound(off, 0, rows), tail = expert_bound(off, num_experts, rows);
    const int64_t n0 = head * pitch16, n1 = (rows - tail) * pitch16;
    uint4* o = static_cast<uint4*>(out);
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * threads + t; i < n0 + n1; i += static_cast<int64_t>(gridDim.x) * threads)
        o[i < n0 ? i : tail * pitch16 + (i - n0)] = make_uint4(0, 0, 0, 0);
}

// Launches `kernel` on as many CTA pairs as fit at once, at most `pairs` of them (the count that fits is cached per device).
struct PairLimit {
    SmemLimitCache smem;
    std::atomic<int> fit[64] = {};
};
template <class Kernel, class... Args>
int launch_pairs(PairLimit& limit, Kernel kernel, int threads, int smem_bytes, int64_t pairs, cudaStream_t stream, const Args&... args) {
    cudaError_t err = limit.smem.ensure(kernel, smem_bytes);
    if (err != cudaSuccess) return static_cast<int>(err);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = dim3(2);
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem_bytes);
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1] = pdl_attribute();
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int dev = 0;
    err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return static_cast<int>(err);
    int n = dev >= 0 && dev < 64 ? limit.fit[dev].load(std::memory_order_relaxed) : 0;
    if (n == 0) {
        // not every SM can always be paired inside its GPC
        if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
            cudaGetLastError();
            n = sm_count_of_current_device() / 2;
        }
        if (dev >= 0 && dev < 64) limit.fit[dev].store(n, std::memory_order_relaxed);
    }
    if (pairs > n) pairs = n;
    cfg.gridDim = dim3(static_cast<unsigned>(2 * (pairs < 1 ? 1 : pairs)));
    cfg.numAttrs = 2;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, args...));
}

// Instruction descriptor of kind::mxf4 / mxf4nvf4: e2m1 (1) at [7,10) and [10,12), N>>3 at [17,23), scale type [23]
// (0 = e4m3, 1 = e8m0), M>>4 at [24,29), bytes of the scale word for B at [4,6) and for A at [29,31): 0 or 2.
template <int FMT>
__device__ __forceinline__ constexpr uint32_t idesc_fp4(uint32_t m, uint32_t n, uint32_t sf_id) {
    return (sf_id << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((FMT == kFp4Mx ? 1u : 0u) << 23) | ((m >> 4) << 24) |
           (sf_id << 29);
}

// Shared-memory matrix without swizzle, 16 bytes wide: groups of 8 rows 128 bytes apart (the 512 bytes of one scale tile)
__device__ __forceinline__ uint64_t desc_scales(uint32_t smem_addr) {
    return static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(128 >> 4) << 32) | (static_cast<uint64_t>(1) << 46);
}

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool live) {  // zeros where not `live`
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
    else
        asm volatile("cp.async.ca.shared.global.L2::128B [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(live ? BYTES : 0), "n"(BYTES) : "memory");
}

// The scale words of rows l, 32 + l, 64 + l, 96 + l that lane l copied to `slot` (its 16 bytes of every 512), in place:
// [row j][K-step i] -> [K-step i][row j], what tcgen05.cp takes to tensor memory.
template <int FMT>
__device__ __forceinline__ void fp4_transpose_scales(uint8_t* slot) {
    if constexpr (FMT == kFp4Nv) {
        const uint4 a = *reinterpret_cast<uint4*>(slot), b = *reinterpret_cast<uint4*>(slot + 512);
        const uint4 c = *reinterpret_cast<uint4*>(slot + 1024), d = *reinterpret_cast<uint4*>(slot + 1536);
        *reinterpret_cast<uint4*>(slot) = make_uint4(a.x, b.x, c.x, d.x);
        *reinterpret_cast<uint4*>(slot + 512) = make_uint4(a.y, b.y, c.y, d.y);
        *reinterpret_cast<uint4*>(slot + 1024) = make_uint4(a.z, b.z, c.z, d.z);
        *reinterpret_cast<uint4*>(slot + 1536) = make_uint4(a.w, b.w, c.w, d.w);
    } else {
        const uint4 a = *reinterpret_cast<uint4*>(slot), b = *reinterpret_cast<uint4*>(slot + 512);
        *reinterpret_cast<uint4*>(slot) = make_uint4(a.x, a.z, b.x, b.z);
        *reinterpret_cast<uint4*>(slot + 512) = make_uint4(a.y, a.w, b.y, b.w);
    }
}
// Where the words of row block j of lane l start before that, beyond the lane's 16 bytes
template <int FMT>
__device__ __forceinline__ uint32_t fp4_scale_at(int j) {
    return FMT == kFp4Nv ? static_cast<uint32_t>(j) * 512u : static_cast<uint32_t>(j >> 1) * 512u + static_cast<uint32_t>(j & 1) * 8u;
}

// 1 / (1 + e^-x) from the fast exponential and division.  Their error bounds, 2 + |1.173 x| and 2 units in the last place, give up to 23
// units of 2^-23 of the result for x = -16, 9 for x = -4, and less than 5 for x > 0, where e^-x is less than half of the sum; 0
// where e^-x overflows.  Rounding act to fp16 is off by up to 2^-11 of it, 4096 of these units, to bf16 by eight times that.
__device__ __forceinline__ float sigmoid_fast(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

// act = silu(g) u with the gradient da of act: dg = da u s (1 + g (1 - s)), du = da g s, s = 1 / (1 + e^-g)
__device__ __forceinline__ void gated_gradients(float da, float g, float u, float& dg, float& du) {
    const float s = sigmoid_fast(g);
    dg = da * u * (s * (1.f + g * (1.f - s)));
    du = da * (g * s);
}

// MN-major tile with 128-byte swizzle: chunks of 64 values along M (or N), each [64 of the contraction][128 bytes]; chunks are
// 8192 bytes apart (leading byte offset), groups of 8 of the contraction 1024 bytes (stride byte offset).
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t smem_addr) {
    return static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(8192 >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
           (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}

// 32 bytes that are read once: a whole sector per thread
__device__ __forceinline__ void ld_nc_f8(const float* p, float* v) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "l"(p));
}

// A box in shared memory (128-byte swizzle) to a matrix; what lies outside of it is not written
__device__ __forceinline__ void tma_store_2d(const void* tmap, uint32_t smem_src, int32_t c0, int32_t c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(tmap)),
                 "r"(smem_src), "r"(c0), "r"(c1)
                 : "memory");
}
__device__ __forceinline__ void tma_store_3d(const void* tmap, uint32_t smem_src, int32_t c0, int32_t c1, int32_t c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(reinterpret_cast<uint64_t>(tmap)),
                 "r"(smem_src), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}

// silu(gate) * up of 32 columns, then scales (two blocks of 16 or one of 32) and codes; `gate` and `up` are raw accumulators.
template <int FMT>
__device__ __forceinline__ void fp4_swiglu32(const uint32_t* gate, const uint32_t* up, float alpha, float out_g, uint4& codes, uint32_t& scales) {
    float act[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        const float g = __uint_as_float(gate[j]) * alpha;
        act[j] = g * sigmoid_fast(g) * (__uint_as_float(up[j]) * alpha);
    }
    uint32_t amax[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 32; ++j) amax[j >> 4] = max(amax[j >> 4], __float_as_uint(act[j]) & 0x7FFFFFFFu);
    if (FMT == kFp4Mx) amax[0] = amax[1] = max(amax[0], amax[1]);
    uint2 c[2];
    uint32_t sc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        Fp4Divisor div;
        sc[h] = fp4_scale<FMT>(amax[h], out_g, __fmul_rn(6.f, out_g), div);
        c[h] = fp4_codes16<FMT>(act + 16 * h, div);
    }
    codes = make_uint4(c[0].x, c[0].y, c[1].x, c[1].y);
    scales = sc[0] | (sc[1] << 8);
}

__device__ __forceinline__ uint32_t pack16(float a, float b, bool fp16) {
    if (fp16) {
        const __half2 t = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&t);
    }
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
}

// Rows of scales of no expert, byte by byte (see zero_loose_rows)
__device__ __forceinline__ void zero_loose_scales(uint8_t* s, int64_t pitch, const int* off, int num_experts, int rows, int t, int threads) {
    const int head = expert_bound(off, 0, rows), tail = expert_bound(off, num_experts, rows);
    const int64_t n0 = head * pitch, n1 = (rows - tail) * pitch;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * threads + t; i < n0 + n1; i += static_cast<int64_t>(gridDim.x) * threads)
        s[i < n0 ? i : tail * pitch + (i - n0)] = 0;
}

}  // namespace cam
