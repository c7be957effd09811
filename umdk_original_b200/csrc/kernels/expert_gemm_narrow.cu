// Row products of the expert-MLP operators for experts with few rows (decode): 4-bit or 16-bit operands, plain or with the
// SwiGLU epilogue, one CTA per tile of 128 rows x 32, 64 or 128 columns.
//
// What bounds these calls is the stream of weights, so the form differs from the CTA pairs (grouped_gemm_fp4.cu,
// grouped_mlp.cu) in what it keeps small:
//   * A tile is narrow enough that there are several for every SM, even where one expert has one row.
//   * The ring of stages is cut for the rows there can be: a stage holds 32, 64 or 128 rows of A beside the weights, and there
//     are as many stages as shared memory holds, so that the weights in flight cover the latency of memory.
//   * A stage of a narrow tile is several K-blocks (128 bytes of every row; `chunks` of them), 16 KiB of weights in all, brought
//     by one TMA instruction: the turn of a stage (two waits, an arrive, a commit) costs each role about 300 cycles, more than
//     the 4 KiB of one K-block of 32 columns take at this SM's share of the memory bandwidth.
//   * No staging: a thread stores 32 columns of its row (64 bytes) from registers.
//   * Scale factors (4-bit): only rows that exist and the tile's own weight rows are brought to tensor memory; with CTA pairs
//     both CTAs need those of all 256 columns.
// The tensor core computes 128 rows whatever there are: a K-block of 128 columns takes 256 cycles for 16 KiB of weights, still
// twice as fast as memory delivers them.
#include "expert_gemm.cuh"

namespace cam {

constexpr int kNwEpiWarps = 8;
constexpr int kNwMaxStages = 24;
constexpr int kNwSfGroup = 4;           // K-blocks whose scales travel together (see grouped_gemm_fp4.cu)
constexpr int kNwScaleSlots = 2 * kNwSfGroup;
constexpr int kNwSfBlock = 4 * 512;     // scales of 128 rows of a K-block
constexpr int kNwSfSlot = 2 * kNwSfBlock;  // of the tile's rows and its weight rows
constexpr uint32_t kNwTmemCols = 512, kNwSfCol0 = 256, kNwSfCols = 32;
static_assert(kNwSfCol0 + kNwScaleSlots * kNwSfCols <= kNwTmemCols, "tensor memory");
constexpr int kNwCtrlBytes = 1024;
static_assert((2 * kNwMaxStages + 8) * 8 + 16 <= kNwCtrlBytes, "barriers");

static __device__ CamStatus g_narrow_status;

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

}  // namespace

template <int KIND, bool SWIGLU>
__global__ void __launch_bounds__(narrow_threads(KIND), 1)
expert_narrow_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const NarrowParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {  // swizzled TMA tiles need it
        if (threadIdx.x == 0) gemm_record_status(&g_narrow_status, CAM_ERR_BAD_INDEX, 4, static_cast<int>(smem_u32(smem) & 1023u));
        return;
    }
    constexpr bool FP4 = KIND != kNarrow16;
    constexpr int SFW = KIND == kFp4Nv ? 4 : 2;  // scale words of a row and K-block
    constexpr int EPI0 = narrow_epi_warp0(KIND);
    const uint32_t ns = static_cast<uint32_t>(p.stages);
    const int width = p.width;
    const int chunks = p.chunks;
    const int a_bytes = p.slot_rows * 128, b_bytes = width * 128;  // of one K-block
    const int a_all = a_bytes * chunks, b_all = b_bytes * chunks;
    const int nstages = (p.kblocks + chunks - 1) / chunks;         // of a tile
    uint8_t* ctrl = smem;
    uint8_t* ring = smem + kNwCtrlBytes;  // stages, each [chunk] rows of A | [chunk] weight rows; behind the last one the scale slots
    uint8_t* sfm = ring + p.stages * p.stage_bytes;
    uint64_t* bar_full = reinterpret_cast<uint64_t*>(ctrl);
    uint64_t* bar_empty = bar_full + kNwMaxStages;
    uint64_t* bar_sf = bar_empty + kNwMaxStages;   // [2]: a group of scale slots is ready
    uint64_t* bar_sfe = bar_sf + 2;                // [2]: the MMAs that read a group's scales have retired
    uint64_t* bar_tfull = bar_sfe + 2;
    uint64_t* bar_tempty = bar_tfull + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_tempty + 2);
    volatile uint32_t* abort_flag = tmem_slot + 1;

    const int warp = static_cast<int>(threadIdx.x) >> 5;
    const uint32_t lane = lane_id();
    const int step = SWIGLU ? width / 2 : width;  // result columns of a tile
    const int n_tiles = (p.n_dim + step - 1) / step;

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
        *abort_flag = 0u;
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, kNwTmemCols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    pdl_wait();
    pdl_release();
    RowWalker<BM> w(p.expert_offsets, p.num_experts, n_tiles, p.rows);
    int e, nt, row0, rows;
    bool ok = true;
    const int tile0 = static_cast<int>(blockIdx.x), tiles_step = static_cast<int>(gridDim.x);

    const uint32_t abort_at = smem_u32(tmem_slot + 1), ring_at = smem_u32(ring);
    const uint32_t full_at = smem_u32(bar_full), sf_at = smem_u32(bar_sf), sfe_at = smem_u32(bar_sfe), empty_at = smem_u32(bar_empty);
    if (warp == 0) {
        // ---------------------------------------------------------------- TMA producer
        const bool leader = elect_one();
        if (leader) {
            prefetch_tensormap(&tmap_a);
            prefetch_tensormap(&tmap_b);
        }
        Ring r;
        uint32_t ready = 1u;  // the first turn of every stage is free
        for (int tile = tile0; w.locate(tile, e, nt, row0, rows); tile += tiles_step) {
            // with several chunks a stage's rows come in one box; otherwise in pieces of 32 rows, those that exist
            const int pieces = chunks > 1 ? 1 : min((rows + 31) / 32, p.slot_rows / 32);
            const uint32_t bytes = static_cast<uint32_t>((chunks > 1 ? a_all : pieces * 4096) + b_all);
            for (int kb = 0; kb < nstages; ++kb) {
                const uint32_t bar = full_at + 8u * r.s, sa = ring_at + r.s * static_cast<uint32_t>(p.stage_bytes);
                if (!ready) mbar_wait_warp(empty_at + 8u * r.s, r.ph ^ 1u, abort_at);
                uint64_t* full = &bar_full[r.s];
                r.next(ns);
                ready = mbar_test(empty_at + 8u * r.s, r.ph ^ 1u);
                if (leader) {
                    mbar_arrive_expect_tx(full, bytes);
                    const int c0 = p.chunked ? 0 : kb * 128, c3 = p.chunked ? kb * chunks : 0;
                    tma_load_5d(sa + static_cast<uint32_t>(a_all), &tmap_b, bar, c0, nt * step, 0, c3, e);
                    for (int i = 0; i < pieces; ++i) tma_load_3d(sa + static_cast<uint32_t>(i) * 4096u, &tmap_a, bar, c0, row0 + i * 32, c3);
                }
                __syncwarp();
            }
        }
        if (leader && *abort_flag) gemm_record_status(&g_narrow_status, CAM_ERR_TIMEOUT_PIPELINE, 0, 0);
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer
        const bool leader = elect_one();
        const uint32_t n = static_cast<uint32_t>(width);
        uint32_t idesc[2];
        if constexpr (FP4) {
            idesc[0] = idesc_fp4<KIND>(BM, 0, 0u) | ((n >> 3) << 17);
            idesc[1] = KIND == kFp4Mx ? idesc_fp4<KIND>(BM, 0, 2u) | ((n >> 3) << 17) : idesc[0];
        } else {
            idesc[0] = idesc[1] = umma_idesc(BM, 0, 1u, p.fp16 ? 0u : 1u) | ((n >> 3) << 17);
        }
        Ring r, groups;
        uint32_t tcount = 0, ready = 0u;
        for (int tile = tile0; w.locate(tile, e, nt, row0, rows); tile += tiles_step, ++tcount) {
            const uint32_t b = tcount & 1u;
            mbar_wait_warp(smem_u32(&bar_tempty[b]), ((tcount >> 1) & 1u) ^ 1u, abort_at);
            for (int kb = 0; kb < nstages; ++kb) {
                // a stage is one or two K-blocks, a group of scales four
                const int k0 = kb * chunks, in_group = k0 % kNwSfGroup;
                const bool group_ends = FP4 && (in_group + chunks == kNwSfGroup || kb == nstages - 1);
                const uint32_t gr = groups.s;
                if (FP4 && in_group == 0) mbar_wait_warp(sf_at + 8u * gr, groups.ph, abort_at);
                if (!ready) mbar_wait_warp(full_at + 8u * r.s, r.ph, abort_at);
                tc_fence_after_sync();
                const uint32_t s = r.s, sa = ring_at + s * static_cast<uint32_t>(p.stage_bytes), sb = sa + static_cast<uint32_t>(a_all);
                r.next(ns);
                ready = mbar_test(full_at + 8u * r.s, r.ph);
                if (group_ends) groups.next(2);
                const int live = min(chunks, p.kblocks - k0);
                if (leader) {
                    for (int c = 0; c < live; ++c) {
                        const uint64_t adesc = umma_desc_k_sw128(sa + static_cast<uint32_t>(c * a_bytes));
                        const uint64_t bdesc = umma_desc_k_sw128(sb + static_cast<uint32_t>(c * b_bytes));
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
                            narrow_mma<KIND>(tmem_base + b * 128u, adesc + 2u * k, bdesc + 2u * k, idesc[k & 1], (kb | c | k) ? 1u : 0u, cs, cs + 4u);
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
        if (leader && *abort_flag) gemm_record_status(&g_narrow_status, CAM_ERR_TIMEOUT_PIPELINE, 1, static_cast<int>(tcount));
    } else if (warp < EPI0) {
        if constexpr (FP4) {
        if (warp >= 4) {
            // ------------------------------------------------------------ scale warps
            // Two for the tile's rows, two for its weight rows, each pair taking groups of four K-blocks in turn; a warp
            // therefore always fills the same half of the slots and sees every turn of it.
            const int weights = warp & 1;
            const uint32_t mine = static_cast<uint32_t>(warp >> 1) & 1u;
            const int words = p.scale_pitch / 4;
            const int w_rows = SWIGLU ? 2 * p.n_dim : p.n_dim;
            const int sub = static_cast<int>(lane) >> 2, piece = static_cast<int>(lane) & 3;  // row of 8, K-block of the group
            uint8_t* slots = sfm + mine * (kNwSfGroup * kNwSfSlot) + weights * kNwSfBlock;
            const uint32_t dst = smem_u32(slots) + static_cast<uint32_t>(piece) * kNwSfSlot + static_cast<uint32_t>(sub) * 16u;
            const int ngroups = (p.kblocks + kNwSfGroup - 1) / kNwSfGroup;
            const int64_t to_up = SWIGLU ? static_cast<int64_t>(p.n_dim - step) * p.scale_pitch : 0;  // from gate row t to up row t - step
            uint32_t count = 0, ph = 0;
            for (int tile = tile0; ok && w.locate(tile, e, nt, row0, rows); tile += tiles_step) {
                const int first = weights ? e * w_rows + nt * step : row0, live = weights ? width : rows;
                const uint8_t* row = (weights ? p.b_scales : p.a_scales) + static_cast<size_t>(first + sub) * p.scale_pitch + piece * (SFW * 4);
                const int64_t jump = weights ? to_up : 0;
                for (int g = 0; g < ngroups; ++g, ++count) {
                    if ((count & 1u) != mine) continue;
                    const bool got = mbar_wait_bounded(&bar_sfe[mine], ph ^ 1u, abort_flag);
                    if (!__all_sync(0xFFFFFFFFu, got)) { ok = false; break; }
                    ph ^= 1u;
                    const uint8_t* from = row + static_cast<size_t>(g) * (kNwSfGroup * SFW * 4);
                    const int left = words - (g * kNwSfGroup + piece) * SFW;  // words of the row that this lane's piece can have
                    if (p.scale_vec) {
                        if (left > 0) {
#pragma unroll
                            for (int i = 0; i < 16; ++i, from += 8 * p.scale_pitch)  // rows 8 i + sub
                                if (8 * i + sub < live) copy_async<SFW * 4>(dst + fp4_scale_at<KIND>(i >> 2) + (i & 3) * 128u, from + (8 * i >= step ? jump : 0), true);
                        }
                    } else {
                        for (int i = 0; i < 16; ++i, from += 8 * p.scale_pitch) {
                            if (8 * i + sub >= live) break;
                            const uint8_t* at = from + (8 * i >= step ? jump : 0);
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
            if (!ok && lane == 0) gemm_record_status(&g_narrow_status, CAM_ERR_TIMEOUT_PIPELINE, 3, static_cast<int>(count));
        }
        }
    } else {
        // ---------------------------------------------------------------- epilogue warps: 32 columns of a row per thread
        const int ew = warp - EPI0;
        const int q = warp & 3;   // TMEM lane quarter this warp may read
        const int cg = ew >> 2;   // column groups cg, cg + 2
        const int r = q * 32 + static_cast<int>(lane);
        const bool fp16 = p.fp16 != 0;
        float a_g = 1.f, out_g = 1.f;
        if constexpr (FP4) {
            if (p.a_gscale != nullptr) a_g = __ldg(p.a_gscale);
            if (p.out_gscale != nullptr) out_g = __ldg(p.out_gscale);
        }
        uint32_t tcount = 0;
        for (int tile = tile0; ok && w.locate(tile, e, nt, row0, rows); tile += tiles_step, ++tcount) {
            const uint32_t b = tcount & 1u;
            const bool valid = r < rows;
            const size_t grow = static_cast<size_t>(row0 + (valid ? r : 0));
            float alpha = a_g;
            if constexpr (FP4) {
                if (p.b_gscale != nullptr) alpha *= __ldg(p.b_gscale + e);
            }
            if (!mbar_wait_bounded(&bar_tfull[b], (tcount >> 1) & 1u, abort_flag, 2000000000ull, 32u)) { ok = false; break; }
            tc_fence_after_sync();
            const uint32_t t0 = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + b * 128u;
            const bool some = q * 32 < rows;  // the same in all lanes: no row of this quarter exists otherwise
            const int groups = (step + 31) / 32;  // groups of 32 result columns
            bool held = true;
            auto hand_back = [&]() {  // what this warp needs of the accumulator is in registers
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar_tempty[b]);
                held = false;
            };
            for (int g = cg; some && g < groups; g += 2) {
                __syncwarp();
                const int c = nt * step + g * 32;
                uint32_t v0[32], v1[32];
                tmem_ld_32x32b_x32(t0 + g * 32, v0);
                if constexpr (SWIGLU) {
                    tmem_ld_32x32b_x32(t0 + (step < 32 ? 0 : step + g * 32), v1);  // width 32: gate and up are halves of v0
                    tc_wait_ld_regs(v1);
                }
                tc_wait_ld_regs(v0);
                if constexpr (SWIGLU && !FP4) {
                    if (step < 32) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) v1[j] = v0[16 + j];
                    }
                }
                if (g + 2 >= groups) hand_back();
                if (!valid) continue;
                if constexpr (FP4 && SWIGLU) {
                    uint4 codes;
                    uint32_t scales;
                    fp4_swiglu32<KIND>(v0, v1, alpha, out_g, codes, scales);
                    if (c < p.n_dim) {  // n_dim is a multiple of 128
                        const size_t at = grow * (p.n_dim / 32) + c / 32;
                        *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + at * 16) = codes;
                        if (KIND == kFp4Nv) *reinterpret_cast<uint16_t*>(p.out_scales + at * 2) = static_cast<uint16_t>(scales);
                        else p.out_scales[at] = static_cast<uint8_t>(scales);
                    }
                } else {
                    const int cols = min(min(32, step), p.n_dim - c);  // a multiple of 8
                    if constexpr (SWIGLU) {
                        if (p.gate_up != nullptr) {
                            const int in_group = min(32, rows - q * 32);
                            // columns c.. are 32-aligned, or half of such a block (width 32)
                            float* gu = p.gate_up + gate_up_at(static_cast<size_t>(row0 + q * 32), in_group, static_cast<int>(lane), p.n_dim, c & ~31) + (c & 31) * in_group;
                            const size_t up = static_cast<size_t>(p.n_dim) * in_group;
#pragma unroll
                            for (int j = 0; j < 32; j += 4) {
                                if (j < cols) {
                                    *reinterpret_cast<uint4*>(gu + j * in_group) = make_uint4(v0[j], v0[j + 1], v0[j + 2], v0[j + 3]);
                                    *reinterpret_cast<uint4*>(gu + up + j * in_group) = make_uint4(v1[j], v1[j + 1], v1[j + 2], v1[j + 3]);
                                }
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const float x = __uint_as_float(v0[j]);
                            v0[j] = __float_as_uint(x * sigmoid_fast(x) * __uint_as_float(v1[j]));
                        }
                    }
                    uint8_t* out = static_cast<uint8_t*>(p.out) + (grow * p.n_dim + c) * 2;
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {
                        if (j < cols) {
                            uint4 o;
                            o.x = pack16(__uint_as_float(v0[j]) * alpha, __uint_as_float(v0[j + 1]) * alpha, fp16);
                            o.y = pack16(__uint_as_float(v0[j + 2]) * alpha, __uint_as_float(v0[j + 3]) * alpha, fp16);
                            o.z = pack16(__uint_as_float(v0[j + 4]) * alpha, __uint_as_float(v0[j + 5]) * alpha, fp16);
                            o.w = pack16(__uint_as_float(v0[j + 6]) * alpha, __uint_as_float(v0[j + 7]) * alpha, fp16);
                            *reinterpret_cast<uint4*>(out + j * 2) = o;
                        }
                    }
                }
            }
            if (held) hand_back();
        }
        if (!ok) gemm_record_status(&g_narrow_status, CAM_ERR_TIMEOUT_PIPELINE, 2, static_cast<int>(tcount));
        const int et = static_cast<int>(threadIdx.x) - EPI0 * 32;
        zero_loose_rows(p.out, (FP4 && SWIGLU) ? p.n_dim / 32 : p.n_dim / 8, p.expert_offsets, p.num_experts, p.rows, et, kNwEpiWarps * 32);
        if constexpr (FP4 && SWIGLU)
            zero_loose_scales(p.out_scales, p.n_dim / fp4_block(KIND), p.expert_offsets, p.num_experts, p.rows, et, kNwEpiWarps * 32);
    }

    // ------------------------------------------------------------------ teardown
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, kNwTmemCols);
    }
}

}  // namespace cam

namespace {

// The MMA reads 128 rows of A from a stage whatever the stage has room for: behind a short one lie weights and scales, and behind
// the last stage this padding.  What it reads there ends in accumulator rows that nobody reads.
int narrow_smem(const cam::NarrowParams* p, bool fp4) {
    const int scales = fp4 ? cam::kNwScaleSlots * cam::kNwSfSlot : 0;
    const int over = (cam::BM - p->slot_rows) * 128 - (p->stage_bytes - p->slot_rows * 128 * p->chunks) - scales;  // from the last chunk's rows
    return cam::kNwCtrlBytes + p->stages * p->stage_bytes + scales + (over > 0 ? over : 0);
}

template <int KIND, bool SWIGLU>
int launch_narrow(const cam::NarrowParams* p, int64_t tiles, const CUtensorMap* ta, const CUtensorMap* tb, cudaStream_t stream) {
    static cam::SmemLimitCache limit;
    const int smem = narrow_smem(p, KIND != cam::kNarrow16);
    const cudaError_t err = limit.ensure(cam::expert_narrow_kernel<KIND, SWIGLU>, smem);
    if (err != cudaSuccess) return static_cast<int>(err);
    const int64_t sms = cam::sm_count_of_current_device();
    const unsigned grid = static_cast<unsigned>(tiles < 1 ? 1 : tiles < sms ? tiles : sms);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1] = {cam::pdl_attribute()};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(static_cast<unsigned>(cam::narrow_threads(KIND)));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, cam::expert_narrow_kernel<KIND, SWIGLU>, *ta, *tb, *p));
}

}  // namespace

extern "C" int cam_launch_expert_gemm_narrow(const cam::NarrowParams* p, int kind, int swiglu, int64_t tiles, const CUtensorMap* ta,
                                             const CUtensorMap* tb, cudaStream_t stream) {
    const bool fp4 = kind != cam::kNarrow16;
    if (p->chunks < 1 || (fp4 && p->chunks > 2) || p->stages < 2 || p->stages > cam::kNwMaxStages || narrow_smem(p, fp4) > 232448 ||
        p->stage_bytes % 1024 != 0)
        return static_cast<int>(cudaErrorInvalidValue);
    if (kind == cam::kFp4Nv) return swiglu ? launch_narrow<cam::kFp4Nv, true>(p, tiles, ta, tb, stream) : launch_narrow<cam::kFp4Nv, false>(p, tiles, ta, tb, stream);
    if (kind == cam::kFp4Mx) return swiglu ? launch_narrow<cam::kFp4Mx, true>(p, tiles, ta, tb, stream) : launch_narrow<cam::kFp4Mx, false>(p, tiles, ta, tb, stream);
    return swiglu ? launch_narrow<cam::kNarrow16, true>(p, tiles, ta, tb, stream) : launch_narrow<cam::kNarrow16, false>(p, tiles, ta, tb, stream);
}

extern "C" int cam_expert_narrow_max_stages(void) { return cam::kNwMaxStages; }

extern "C" int cam_narrow_status(CamStatus* out) { return static_cast<int>(cudaMemcpyFromSymbol(out, cam::g_narrow_status, sizeof(CamStatus))); }
