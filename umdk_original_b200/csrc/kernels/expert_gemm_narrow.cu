// Row products of the expert-MLP operators for experts with few rows (decode, small training batches): 4-bit or 16-bit operands,
// plain or with the SwiGLU epilogue; in 16 bits also the backward products dact and dx (formulas in grouped_mlp.cu), whose weights are
// contracted over their rows and read in the tensor core's MN-major form.  One CTA computes 128 weight rows x the rows of an expert (at
// most 32, 64 or 128 of them).
//
// What bounds these calls is the stream of weights, so the form differs from the CTA pairs (grouped_gemm_fp4.cu,
// grouped_mlp.cu) in what it spends per weight byte:
//   * The weights are the M operand of the tensor core and the rows its N operand, in steps of 16.  An MMA then takes as long as
//     there are rows: 67 cycles up to 32 of them, about twice that for 128, the time it takes for any number of rows when the rows
//     are the M operand.  A K-block (128 bytes of every row) is 16 KiB of weights and four MMAs; memory delivers it in 740 cycles.
//   * A stage of the ring is one or two K-blocks, brought by one TMA instruction for the weights and one for the rows: the turn of
//     a stage costs each role about 300 cycles, whatever it holds.
//   * Where there are fewer tiles than SMs, a cluster of 2 or 4 CTAs shares the K-blocks of a tile.  Each CTA stores its sums
//     in the staging area of the CTA that finishes the row (distributed shared memory), which adds them up in the CTAs' order.
// The accumulator has a weight row per lane and a row of the expert per column; it goes through shared memory as fp32, and the
// threads that pick it up again own 8 or 16 neighbouring columns of a row each.
//
// Measured (one call, L2 cold, launch included): 32 experts of 32 rows, nvfp4, 7168 -> 2 x 2048 with SwiGLU 111 us (4.9 TB/s), 29 of 35
// rows, 2048 -> 7168 62 us (4.2 TB/s); mxfp4 100 and 57 us; 8 experts of one row 43 and 29 us; 16 experts of 32 rows in 16 bits, 4096 -> 2
// x 1024 50 us, 1024 -> 4096 28 us.  Left out one at a time, the weights, the scales and the MMAs each save 10 to 15 %, all three half:
// no single unit is saturated, the short tiles (8 to 28 K-blocks) leave the turns of the stages, the start and the last wave.
// Scales stored to tensor memory from registers, loaded a group ahead: no faster (62 us), and 10 % slower for one row per expert.
#include "expert_gemm.cuh"

namespace cam {

constexpr int kNwEpiWarps = 8, kNwEpiThreads = kNwEpiWarps * 32;
constexpr int kNwMaxStages = 12;
constexpr int kNwSfGroup = 4;           // K-blocks whose scales travel together (see grouped_gemm_fp4.cu)
constexpr int kNwScaleSlots = 2 * kNwSfGroup;
constexpr int kNwSfBlock = 4 * 512;     // scales of 128 rows of a K-block
constexpr int kNwSfSlot = 2 * kNwSfBlock;  // of the weight rows and of the expert's rows
constexpr int kNwPitch = 132;           // floats between the staged rows
constexpr uint32_t kNwTmemCols = 512, kNwSfCol0 = 256, kNwSfCols = 32;
static_assert(kNwSfCol0 + kNwScaleSlots * kNwSfCols <= kNwTmemCols, "tensor memory");
constexpr int kNwCtrlBytes = 1024;
static_assert((2 * kNwMaxStages + 10) * 8 + 16 <= kNwCtrlBytes, "barriers");

namespace {

template <int KIND>
__device__ __forceinline__ void narrow_mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate,
                                           uint32_t sfa, uint32_t sfb) {
    if constexpr (KIND == kFp4Nv)
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n"
            "}\n" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb) : "memory");
    else if constexpr (KIND == kFp4Mx)
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n"
            "}\n" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb) : "memory");
    else
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
            "}\n" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

__device__ __forceinline__ void tc_copy_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t smem_dst, const void* tmap, uint32_t bar, int32_t c0, int32_t c1, int32_t c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
__device__ __forceinline__ void tma_load_5d(uint32_t smem_dst, const void* tmap, uint32_t bar, int32_t c0, int32_t c1, int32_t c2, int32_t c3, int32_t c4) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
        ::"r"(smem_dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
        : "memory");
}

__host__ __device__ constexpr int narrow_epi_warp0(int kind) { return kind == kNarrow16 ? 4 : 8; }
__host__ __device__ constexpr int narrow_threads(int kind) { return (narrow_epi_warp0(kind) + kNwEpiWarps) * 32; }

// Barriers between the CTAs of a cluster that guard ordinary accesses to each other's shared memory
__device__ __forceinline__ void arrive_release_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool wait_acquire_cluster(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag) {
    for (uint32_t n = 0; n < kWaitPolls; ++n) {
        uint32_t ok;
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
        if ((n & 255u) == 255u && *abort_flag) return false;
    }
    *abort_flag = 1u;
    return false;
}
__device__ __forceinline__ void st_cluster_f32(uint32_t cluster_addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}

// Tiles of `tm` rows x n_tiles columns, see RowWalker
struct TallWalker {
    const int* off;
    int num_experts, n_tiles, rows_total, tm;
    int e = 0, base = 0;
    __device__ TallWalker(const int* o, int ne, int nt, int rt, int t) : off(o), num_experts(ne), n_tiles(nt), rows_total(rt), tm(t) {}
    __device__ bool locate(int tile, int& e_out, int& nt, int& row0, int& rows) {
        while (e < num_experts) {
            const int first = expert_bound(off, e, rows_total);
            const int cnt = max(expert_bound(off, e + 1, rows_total) - first, 0);
            const int tiles = ((cnt + tm - 1) / tm) * n_tiles;
            if (tile < base + tiles) {
                const int local = tile - base, mt = local / n_tiles;
                nt = local - mt * n_tiles;
                row0 = first + mt * tm;
                rows = min(tm, cnt - mt * tm);
                e_out = e;
                return true;
            }
            base += tiles;
            ++e;
        }
        return false;
    }
};

}  // namespace

template <int KIND, int FORM>
__global__ void __launch_bounds__(narrow_threads(KIND), 1)
expert_narrow_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const NarrowParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {  // swizzled TMA tiles need it; the same in all CTAs of a cluster
        if (threadIdx.x == 0) record_status(p.status, CAM_ERR_BAD_INDEX, 4, static_cast<int>(smem_u32(smem) & 1023u));
        return;
    }
    constexpr bool FP4 = KIND != kNarrow16, SWIGLU = FORM == kNarrowSwiglu, DACT = FORM == kNarrowDact;
    constexpr bool W_MN = DACT || FORM == kNarrowByRows;  // the weights' contraction index is their row index in memory
    constexpr int SFW = KIND == kFp4Nv ? 4 : 2;  // scale words of a row and K-block
    constexpr int EPI0 = narrow_epi_warp0(KIND);
    constexpr int STEP = SWIGLU ? 64 : 128;      // result columns of a tile: 64 gate and 64 up rows, or 128 rows
    const uint32_t ns = static_cast<uint32_t>(p.stages);
    const int chunks = p.chunks, split = p.split, shift = 31 - __clz(split);  // a power of two
    const int a_bytes = p.slot_rows * 128, a_all = a_bytes * chunks;  // rows of a K-block, of a stage
    constexpr int kWBytes = 128 * 128;
    uint8_t* ctrl = smem;
    uint8_t* ring = smem + kNwCtrlBytes;  // stages, each [chunk] weight rows | [chunk] rows
    uint8_t* sfm = ring + p.stages * p.stage_bytes;  // 4-bit: scale slots
    float* stg = reinterpret_cast<float*>(sfm + (FP4 ? kNwScaleSlots * kNwSfSlot : 0));  // [slot_rows][kNwPitch]
    uint64_t* bar_full = reinterpret_cast<uint64_t*>(ctrl);
    uint64_t* bar_empty = bar_full + kNwMaxStages;
    uint64_t* bar_sf = bar_empty + kNwMaxStages;   // [2]: a group of scale slots is ready
    uint64_t* bar_sfe = bar_sf + 2;                // [2]: the MMAs that read a group's scales have retired
    uint64_t* bar_tfull = bar_sfe + 2;             // [2]
    uint64_t* bar_tempty = bar_tfull + 2;          // [2]
    uint64_t* bar_part = bar_tempty + 2;           // cluster: every CTA has staged its sums
    uint64_t* bar_free = bar_part + 1;             // cluster: every CTA has read this one's
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_free + 1);
    volatile uint32_t* abort_flag = tmem_slot + 1;

    const int warp = static_cast<int>(threadIdx.x) >> 5;
    const uint32_t lane = lane_id();
    const int rank = static_cast<int>(cluster_cta_rank());
    const int n_tiles = (p.n_dim + STEP - 1) / STEP;
    // this CTA's K-blocks: units of a group of scales, or of a stage
    const int unit = FP4 ? kNwSfGroup : chunks, units = (p.kblocks + unit - 1) / unit;
    const int k_lo = ((rank * units) >> shift) * unit;
    const int k_hi = min(p.kblocks, (((rank + 1) * units) >> shift) * unit);
    const int nstages = (k_hi - k_lo + chunks - 1) / chunks;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < ns; ++s) {
            mbar_init(&bar_full[s], 1);
            mbar_init(&bar_empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bar_sf[b], 2);
            mbar_init(&bar_sfe[b], 1);
            mbar_init(&bar_tfull[b], 1);
            mbar_init(&bar_tempty[b], kNwEpiWarps);
        }
        mbar_init(bar_part, static_cast<uint32_t>(split));
        mbar_init(bar_free, static_cast<uint32_t>(split));
        *abort_flag = 0u;
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, kNwTmemCols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    if (split > 1) cluster_sync_all();  // all CTAs' barriers are initialised before anything signals them
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    pdl_wait();
    pdl_release();
    TallWalker w(p.expert_offsets, p.num_experts, n_tiles, p.rows, p.slot_rows);
    int e, nt, row0, rows;
    bool ok = true;
    const int tile0 = static_cast<int>(blockIdx.x) >> shift, tiles_step = static_cast<int>(gridDim.x) >> shift;

    const uint32_t abort_at = smem_u32(tmem_slot + 1), ring_at = smem_u32(ring);
    const uint32_t full_at = smem_u32(bar_full), sf_at = smem_u32(bar_sf), empty_at = smem_u32(bar_empty);
    if (warp == 0) {
        // ---------------------------------------------------------------- TMA producer
        const bool leader = elect_one();
        if (leader) {
            prefetch_tensormap(&tmap_a);
            prefetch_tensormap(&tmap_b);
        }
        Ring r;
        uint32_t ready = 1u;  // the first turn of every stage is free
        for (int tile = tile0; !aborted(abort_flag) && w.locate(tile, e, nt, row0, rows); tile += tiles_step) {
            // with two chunks a stage's rows come in one box; otherwise in pieces of 32 rows, those that exist
            const int pieces = chunks > 1 ? 1 : (rows + 31) / 32;
            const uint32_t bytes = static_cast<uint32_t>((chunks > 1 ? a_all : pieces * 4096) + kWBytes * chunks);
            for (int st = 0; st < nstages; ++st) {
                const uint32_t bar = full_at + 8u * r.s, sw = ring_at + r.s * static_cast<uint32_t>(p.stage_bytes);
                if (!ready) mbar_wait_warp(empty_at + 8u * r.s, r.ph ^ 1u, abort_at);
                uint64_t* full = &bar_full[r.s];
                r.next(ns);
                ready = mbar_test(empty_at + 8u * r.s, r.ph ^ 1u);
                if (leader) {
                    const int k = k_lo + st * chunks;
                    mbar_arrive_expect_tx(full, bytes);
                    const int c0 = p.chunked ? 0 : k * 128, c3 = p.chunked ? k : 0;
                    if constexpr (W_MN) {
                        for (int i = 0; i < 2 * chunks; ++i)  // [64 of the contraction][64 values]; what lies outside comes as zeros
                            tma_load_3d(sw + static_cast<uint32_t>(i) * 8192u, &tmap_b, bar, (nt * STEP + (i & 1) * 64) * 2, (k + (i >> 1)) * 64, e);
                    } else {
                        tma_load_5d(sw, &tmap_b, bar, c0, nt * STEP, 0, c3, e);
                    }
                    const uint32_t sr = sw + static_cast<uint32_t>(kWBytes * chunks);
                    for (int i = 0; i < pieces; ++i) tma_load_3d(sr + static_cast<uint32_t>(i) * 4096u, &tmap_a, bar, c0, row0 + i * 32, c3);
                }
                __syncwarp();
            }
        }
        if (leader && *abort_flag) record_status(p.status, CAM_ERR_TIMEOUT_PIPELINE, 0, 0);
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer
        const bool leader = elect_one();
        Ring r, groups;
        uint32_t tcount = 0, ready = 0u;
        for (int tile = tile0; !aborted(abort_flag) && w.locate(tile, e, nt, row0, rows); tile += tiles_step, ++tcount) {
            const uint32_t n = static_cast<uint32_t>((rows + 15) & ~15);
            uint32_t idesc[2];
            if constexpr (FP4) {
                idesc[0] = idesc_fp4<KIND>(BM, 0, 0u) | ((n >> 3) << 17);
                idesc[1] = KIND == kFp4Mx ? idesc_fp4<KIND>(BM, 0, 2u) | ((n >> 3) << 17) : idesc[0];
            } else {
                idesc[0] = idesc[1] = umma_idesc(BM, 0, 1u, p.fp16 ? 0u : 1u) | ((n >> 3) << 17) | (W_MN ? 1u << 15 : 0u);
            }
            const uint32_t b = tcount & 1u;
            mbar_wait_warp(smem_u32(&bar_tempty[b]), ((tcount >> 1) & 1u) ^ 1u, abort_at);
            for (int st = 0; st < nstages; ++st) {
                // a stage is one or two K-blocks, a group of scales four
                const int in_group = (st * chunks) % kNwSfGroup;
                const bool group_ends = FP4 && (in_group + chunks == kNwSfGroup || st == nstages - 1);
                const uint32_t gr = groups.s;
                if (FP4 && in_group == 0) mbar_wait_warp(sf_at + 8u * gr, groups.ph, abort_at);
                if (!ready) mbar_wait_warp(full_at + 8u * r.s, r.ph, abort_at);
                tc_fence_after_sync();
                const uint32_t s = r.s, sw = ring_at + s * static_cast<uint32_t>(p.stage_bytes), sr = sw + static_cast<uint32_t>(kWBytes * chunks);
                r.next(ns);
                ready = mbar_test(full_at + 8u * r.s, r.ph);
                if (group_ends) groups.next(2);
                const int live = min(chunks, k_hi - k_lo - st * chunks);
                if (leader) {
                    for (int c = 0; c < live; ++c) {
                        const uint32_t wat = sw + static_cast<uint32_t>(c * kWBytes);
                        const uint64_t wdesc = W_MN ? umma_desc_mn_sw128(wat) : umma_desc_k_sw128(wat);
                        const uint64_t rdesc = umma_desc_k_sw128(sr + static_cast<uint32_t>(c * a_bytes));
                        const uint32_t slot = gr * kNwSfGroup + static_cast<uint32_t>(in_group + c), sf = tmem_base + kNwSfCol0 + slot * kNwSfCols;
                        if constexpr (FP4) {
                            const uint32_t sfs = smem_u32(sfm) + slot * kNwSfSlot;
#pragma unroll
                            for (int k = 0; k < SFW; ++k) {
                                tc_copy_scales(sf + 8u * k, desc_scales(sfs + k * 512));
                                tc_copy_scales(sf + 8u * k + 4u, desc_scales(sfs + kNwSfBlock + k * 512));
                            }
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t cs = sf + 8u * (KIND == kFp4Mx ? k >> 1 : k);
                            narrow_mma<KIND>(tmem_base + b * 128u, wdesc + (W_MN ? 128u : 2u) * k, rdesc + 2u * k, idesc[k & 1], (st | c | k) ? 1u : 0u, cs, cs + 4u);
                        }
                    }
                    tc_commit(&bar_empty[s]);
                    if (group_ends) tc_commit(&bar_sfe[gr]);  // shared and tensor memory of the group's scales are free
                }
                __syncwarp();
            }
            if (leader) tc_commit(&bar_tfull[b]);
            __syncwarp();
        }
        if (leader && *abort_flag) record_status(p.status, CAM_ERR_TIMEOUT_PIPELINE, 1, static_cast<int>(tcount));
    } else if (warp < EPI0) {
        if constexpr (FP4) {
        if (warp >= 4) {
            // ------------------------------------------------------------ scale warps
            // Two for the weight rows, two for the expert's rows, each pair taking groups of four K-blocks in turn; a warp
            // therefore always fills the same half of the slots and sees every turn of it.
            const int which = warp & 1;  // 0: weights, 1: rows
            const uint32_t mine = static_cast<uint32_t>(warp >> 1) & 1u;
            const int words = p.scale_pitch / 4;
            const int w_rows = SWIGLU ? 2 * p.n_dim : p.n_dim;
            const int sub = static_cast<int>(lane) >> 2, piece = static_cast<int>(lane) & 3;  // row of 8, K-block of the group
            uint8_t* slots = sfm + mine * (kNwSfGroup * kNwSfSlot) + which * kNwSfBlock;
            const uint32_t dst = smem_u32(slots) + static_cast<uint32_t>(piece) * kNwSfSlot + static_cast<uint32_t>(sub) * 16u;
            // from gate row t to up row t - 64
            const int64_t jump = SWIGLU && which == 0 ? static_cast<int64_t>(p.n_dim - STEP) * p.scale_pitch : 0;
            uint32_t count = 0, ph = 0;
            for (int tile = tile0; ok && w.locate(tile, e, nt, row0, rows); tile += tiles_step) {
                const int first = which == 0 ? e * w_rows + nt * STEP : row0;
                const int live = which == 0 ? 128 : rows;  // n_dim is a multiple of 128: all weight rows exist
                const uint8_t* row = (which == 0 ? p.b_scales : p.a_scales) + static_cast<size_t>(first + sub) * p.scale_pitch + piece * (SFW * 4);
                for (int k = k_lo; k < k_hi; k += kNwSfGroup, ++count) {
                    if ((count & 1u) != mine) continue;
                    const bool got = mbar_wait_bounded(&bar_sfe[mine], ph ^ 1u, abort_flag);
                    if (!__all_sync(0xFFFFFFFFu, got)) { ok = false; break; }
                    ph ^= 1u;
                    const uint8_t* from = row + static_cast<size_t>(k) * (SFW * 4);
                    const int left = words - (k + piece) * SFW;  // words of the row that this lane's piece can have
                    if (p.scale_vec) {
                        if (left > 0) {
#pragma unroll
                            for (int i = 0; i < 16; ++i, from += 8 * p.scale_pitch)  // rows 8 i + sub
                                if (8 * i + sub < live) copy_async<SFW * 4>(dst + fp4_scale_at<KIND>(i >> 2) + (i & 3) * 128u, from + (8 * i >= STEP ? jump : 0), true);
                        }
                    } else {
                        for (int i = 0; i < 16; ++i, from += 8 * p.scale_pitch) {
                            if (8 * i + sub >= live) break;
                            const uint8_t* at = from + (8 * i >= STEP ? jump : 0);
#pragma unroll
                            for (int j = 0; j < SFW; ++j)
                                copy_async<4>(dst + fp4_scale_at<KIND>(i >> 2) + (i & 3) * 128u + j * 4u, j < left ? at + j * 4 : p.a_scales, j < left);
                        }
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    __syncwarp();  // the words a lane transposes were copied by others
#pragma unroll
                    for (int c = 0; c < kNwSfGroup; ++c) fp4_transpose_scales<KIND>(slots + c * kNwSfSlot + lane * 16u);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bar_sf[mine]);
                }
            }
            if (!ok && lane == 0) record_status(p.status, CAM_ERR_TIMEOUT_PIPELINE, 3, static_cast<int>(count));
        }
        }
    } else {
        // ---------------------------------------------------------------- epilogue
        const int q = warp & 3;             // TMEM lane quarter this warp may read
        const int cg = (warp - EPI0) >> 2;  // rows 32 cg .., 64 + 32 cg ..
        const int f = q * 32 + static_cast<int>(lane);                 // weight row of the tile
        const int te = static_cast<int>(threadIdx.x) - EPI0 * 32;      // 0..255
        const bool fp16 = p.fp16 != 0;
        float a_g = 1.f, out_g = 1.f;
        if constexpr (FP4) {
            if (p.a_gscale != nullptr) a_g = __ldg(p.a_gscale);
            if (p.out_gscale != nullptr) out_g = __ldg(p.out_gscale);
        }
        uint32_t tcount = 0;
        // Staged row t, t = rank, rank + split, ... of the tile: `split` copies, one from each CTA, slot_rows / split rows apart.
        // `n4` groups of 4 floats from column c on, summed.
        const int copy_rows = p.slot_rows >> shift;
        auto gather = [&](float* v, int n4, int t, int c) {
            const float* at = stg + (t >> shift) * kNwPitch + c;
            for (int i = 0; i < n4; ++i) *reinterpret_cast<float4*>(v + 4 * i) = *reinterpret_cast<const float4*>(at + 4 * i);
            for (int d = 1; d < split; ++d) {
                at += copy_rows * kNwPitch;
                for (int i = 0; i < n4; ++i) {
                    const float4 x = *reinterpret_cast<const float4*>(at + 4 * i);
                    v[4 * i] += x.x; v[4 * i + 1] += x.y; v[4 * i + 2] += x.z; v[4 * i + 3] += x.w;
                }
            }
        };
        for (int tile = tile0; ok && w.locate(tile, e, nt, row0, rows); tile += tiles_step, ++tcount) {
            const uint32_t b = tcount & 1u;
            float alpha = a_g;
            if constexpr (FP4) {
                if (p.b_gscale != nullptr) alpha *= __ldg(p.b_gscale + e);
            }
            bool got = mbar_wait_bounded(&bar_tfull[b], (tcount >> 1) & 1u, abort_flag, 2000000000ull, 32u);
            // the staging areas of the tile before have been read, in all CTAs of the cluster
            if (split > 1 && tcount > 0) got = wait_acquire_cluster(bar_free, (tcount - 1u) & 1u, abort_flag) && got;
            if (!named_bar_and(1, kNwEpiThreads, got)) { ok = false; break; }
            tc_fence_after_sync();
            const uint32_t t0 = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + b * 128u;
            for (int c0 = cg * 32; c0 < rows; c0 += 64) {
                uint32_t v[32];
                tmem_ld_32x32b_x32(t0 + static_cast<uint32_t>(c0), v);
                tc_wait_ld_regs(v);
                if (split == 1) {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (c0 + j < rows) stg[(c0 + j) * kNwPitch + f] = __uint_as_float(v[j]);
                } else {
                    const float* mine = stg + rank * copy_rows * kNwPitch + f;
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (c0 + j < rows)
                            st_cluster_f32(map_to_cta(mine + ((c0 + j) >> shift) * kNwPitch, static_cast<uint32_t>((c0 + j) & (split - 1))), __uint_as_float(v[j]));
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_tempty[b]);
            named_bar_sync(1, kNwEpiThreads);
            if (split > 1) {
                if (te < split) arrive_release_cluster(map_to_cta(bar_part, static_cast<uint32_t>(te)));
                got = wait_acquire_cluster(bar_part, tcount & 1u, abort_flag);
                if (!named_bar_and(1, kNwEpiThreads, got)) { ok = false; break; }
            }
            // rows rank, rank + split, ... of the tile are this CTA's
            const int my_rows = (rows - rank + split - 1) >> shift;
            if constexpr (FP4 && SWIGLU) {
                // 16 columns of a row per thread: an nvfp4 block, or half of an mxfp4 block
                for (int i = te; (i & ~31) < my_rows * 4; i += kNwEpiThreads) {  // whole warps stay together
                    const int t = ((i >> 2) << shift) + rank, ch = i & 3;
                    const bool live = t < rows;
                    float g[16], u[16];
                    gather(g, 4, live ? t : 0, ch * 16);
                    gather(u, 4, live ? t : 0, 64 + ch * 16);
                    uint32_t amax = 0u;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float x = g[j] * alpha;
                        g[j] = x * sigmoid_fast(x) * (u[j] * alpha);
                        amax = max(amax, __float_as_uint(g[j]) & 0x7FFFFFFFu);
                    }
                    if (KIND == kFp4Mx) amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
                    Fp4Divisor div;
                    const uint32_t code = fp4_scale<KIND>(amax, out_g, __fmul_rn(6.f, out_g), div);
                    const uint2 codes = fp4_codes16<KIND>(g, div);
                    if (live) {
                        const size_t at = static_cast<size_t>(row0 + t) * (p.n_dim / 16) + nt * 4 + ch;  // in units of 16 columns
                        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.out) + at * 8) = codes;
                        if (KIND == kFp4Nv) p.out_scales[at] = static_cast<uint8_t>(code);
                        else if ((ch & 1) == 0) p.out_scales[at >> 1] = static_cast<uint8_t>(code);
                    }
                }
            } else {
                constexpr int PER = STEP / 8;  // threads per row, 8 columns each
                for (int i = te; i < my_rows * PER; i += kNwEpiThreads) {
                    const int t = ((i / PER) << shift) + rank, ch = i % PER, c = nt * STEP + ch * 8;
                    if (c >= p.n_dim) continue;  // n_dim is a multiple of 8
                    float v[8];
                    gather(v, 2, t, ch * 8);
                    if constexpr (DACT) {
                        const size_t at = static_cast<size_t>(row0 + t) * (2 * static_cast<size_t>(p.n_dim)) + c;
                        float g[8], u[8], dg[8], du[8];
                        ld_nc_f8(p.gate_up + at, g);
                        ld_nc_f8(p.gate_up + at + p.n_dim, u);
#pragma unroll
                        for (int j = 0; j < 8; ++j) gated_gradients(v[j], g[j], u[j], dg[j], du[j]);
                        uint16_t* o = static_cast<uint16_t*>(p.out) + at;
                        *reinterpret_cast<uint4*>(o) = make_uint4(pack16(dg[0], dg[1], fp16), pack16(dg[2], dg[3], fp16), pack16(dg[4], dg[5], fp16), pack16(dg[6], dg[7], fp16));
                        *reinterpret_cast<uint4*>(o + p.n_dim) = make_uint4(pack16(du[0], du[1], fp16), pack16(du[2], du[3], fp16), pack16(du[4], du[5], fp16), pack16(du[6], du[7], fp16));
                        continue;
                    }
                    if constexpr (SWIGLU) {
                        float u[8];
                        gather(u, 2, t, 64 + ch * 8);
                        if (p.gate_up != nullptr) {
                            float* gu = p.gate_up + static_cast<size_t>(row0 + t) * (2 * static_cast<size_t>(p.n_dim)) + c;
#pragma unroll
                            for (int j = 0; j < 8; j += 4) {
                                *reinterpret_cast<float4*>(gu + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                                *reinterpret_cast<float4*>(gu + p.n_dim + j) = make_float4(u[j], u[j + 1], u[j + 2], u[j + 3]);
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = v[j] * sigmoid_fast(v[j]) * u[j];
                    }
                    uint4 o;
                    o.x = pack16(v[0] * alpha, v[1] * alpha, fp16);
                    o.y = pack16(v[2] * alpha, v[3] * alpha, fp16);
                    o.z = pack16(v[4] * alpha, v[5] * alpha, fp16);
                    o.w = pack16(v[6] * alpha, v[7] * alpha, fp16);
                    *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + (static_cast<size_t>(row0 + t) * p.n_dim + c) * 2) = o;
                }
            }
            if (split > 1) {
                named_bar_sync(1, kNwEpiThreads);
                if (te < split) arrive_release_cluster(map_to_cta(bar_free, static_cast<uint32_t>(te)));
            }
        }
        if (!ok && te == 0) record_status(p.status, CAM_ERR_TIMEOUT_PIPELINE, 2, static_cast<int>(tcount));
        if constexpr (!DACT)  // dgu of rows of no expert is read by nothing
            zero_loose_rows(p.out, (FP4 && SWIGLU) ? p.n_dim / 32 : p.n_dim / 8, p.expert_offsets, p.num_experts, p.rows, te, kNwEpiThreads);
        if constexpr (FP4 && SWIGLU)
            zero_loose_scales(p.out_scales, p.n_dim / fp4_block(KIND), p.expert_offsets, p.num_experts, p.rows, te, kNwEpiThreads);
    }

    // ------------------------------------------------------------------ teardown
    abort_drain(abort_flag);
    tc_fence_before_sync();
    __syncthreads();
    if (split > 1) cluster_sync_all();  // another CTA may still read this one's staging area or signal its barriers
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, kNwTmemCols);
    }
}

}  // namespace cam

namespace {

int narrow_smem(const cam::NarrowParams* p, bool fp4) {
    return cam::kNwCtrlBytes + p->stages * p->stage_bytes + (fp4 ? cam::kNwScaleSlots * cam::kNwSfSlot : 0) + p->slot_rows * cam::kNwPitch * 4;
}

template <int KIND, int FORM>
int launch_narrow(const cam::NarrowParams* p, int64_t tiles, const CUtensorMap* ta, const CUtensorMap* tb, cudaStream_t stream) {
    static cam::SmemLimitCache limit;
    const int smem = narrow_smem(p, KIND != cam::kNarrow16);
    const cudaError_t err = limit.ensure(cam::expert_narrow_kernel<KIND, FORM>, smem);
    if (err != cudaSuccess) return static_cast<int>(err);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2] = {cam::pdl_attribute(), {}};
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(p->split);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    const int64_t most = cam::sm_count_of_current_device() / p->split;
    cfg.gridDim = dim3(static_cast<unsigned>((tiles < 1 ? 1 : tiles < most ? tiles : most) * p->split));
    cfg.blockDim = dim3(static_cast<unsigned>(cam::narrow_threads(KIND)));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = p->split > 1 ? 2 : 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, cam::expert_narrow_kernel<KIND, FORM>, *ta, *tb, *p));
}

}  // namespace

extern "C" int cam_launch_expert_gemm_narrow(const cam::NarrowParams* p, int kind, int form, int64_t tiles, const CUtensorMap* ta,
                                             const CUtensorMap* tb, cudaStream_t stream) {
    const bool fp4 = kind != cam::kNarrow16;
    const int unit = fp4 ? cam::kNwSfGroup : p->chunks;
    if (p->chunks < 1 || p->chunks > 2 || p->stages < 2 || p->stages > cam::kNwMaxStages || narrow_smem(p, fp4) > 232448 ||
        p->stage_bytes % 1024 != 0 || (p->split != 1 && p->split != 2 && p->split != 4) || p->split > (p->kblocks + unit - 1) / unit)
        return static_cast<int>(cudaErrorInvalidValue);
    switch (kind * 4 + form) {
        case cam::kFp4Nv * 4 + cam::kNarrowPlain: return launch_narrow<cam::kFp4Nv, cam::kNarrowPlain>(p, tiles, ta, tb, stream);
        case cam::kFp4Nv * 4 + cam::kNarrowSwiglu: return launch_narrow<cam::kFp4Nv, cam::kNarrowSwiglu>(p, tiles, ta, tb, stream);
        case cam::kFp4Mx * 4 + cam::kNarrowPlain: return launch_narrow<cam::kFp4Mx, cam::kNarrowPlain>(p, tiles, ta, tb, stream);
        case cam::kFp4Mx * 4 + cam::kNarrowSwiglu: return launch_narrow<cam::kFp4Mx, cam::kNarrowSwiglu>(p, tiles, ta, tb, stream);
        case cam::kNarrow16 * 4 + cam::kNarrowPlain: return launch_narrow<cam::kNarrow16, cam::kNarrowPlain>(p, tiles, ta, tb, stream);
        case cam::kNarrow16 * 4 + cam::kNarrowSwiglu: return launch_narrow<cam::kNarrow16, cam::kNarrowSwiglu>(p, tiles, ta, tb, stream);
        case cam::kNarrow16 * 4 + cam::kNarrowDact: return launch_narrow<cam::kNarrow16, cam::kNarrowDact>(p, tiles, ta, tb, stream);
        case cam::kNarrow16 * 4 + cam::kNarrowByRows: return launch_narrow<cam::kNarrow16, cam::kNarrowByRows>(p, tiles, ta, tb, stream);
    }
    return static_cast<int>(cudaErrorInvalidValue);
}

extern "C" int cam_expert_narrow_max_stages(void) { return cam::kNwMaxStages; }

extern "C" int cam_expert_narrow_fixed_smem(int fp4, int slot_rows) {
    return cam::kNwCtrlBytes + (fp4 ? cam::kNwScaleSlots * cam::kNwSfSlot : 0) + slot_rows * cam::kNwPitch * 4;
}
