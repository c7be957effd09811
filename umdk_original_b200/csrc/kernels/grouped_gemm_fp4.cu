// Grouped product of 4-bit operands (nvfp4 / mxfp4, ../common/fp4.cuh) on CTA pairs, for the rows of every expert:
//   y[r, n] = a_g w_g[e] sum_k (a_q a_s)[r, k] (w_q w_s)[e, n, k]
// and the first product of an expert MLP, whose epilogue forms silu(gate) * up and writes it back as 4-bit rows.
//
// The tensor core multiplies e2m1 values and applies the block scales itself (kind::mxf4nvf4 with 16 values per scale,
// kind::mxf4 with 32), so a tile is a loop over K-blocks of 256 values (128 bytes of a row).  A pair of CTAs computes 256
// rows x 256 columns: each holds its 128 rows of A and HALF of the weight tile, one CTA issues the MMAs of both.
//
// Scales stay in memory as the quantiser wrote them, row by row; the tensor core wants them in tensor memory as
// [32 lanes][4 words] per 128 rows and 64 values (word j of lane l: row 32 j + l).  Three warps per CTA (its rows, the lower and
// the upper 128 weight rows) bring them there, four K-blocks at a time: 64 bytes of a row are copied by four lanes with cp.async,
// each to the slot of its K-block, then lane l transposes the 4 x 4 words of rows l, 32 + l, 64 + l, 96 + l of each K-block in
// place and the warp raises the group's barrier.  The MMA issuer moves a slot into tensor memory with tcgen05.cp directly in
// front of the MMAs that read it.  Four K-blocks at a time, because these warps are paced by the rows
// they touch: one K-block at a time (16 bytes of every row) took them 1070 cycles where the MMAs take 512.
//
// Measured (one call, L2 cold): 16 experts of 1024 rows, 7168 -> 2 x 2048 with SwiGLU: nvfp4 240 us (4.0 PFLOP/s), mxfp4 184 us (5.2);
// 32 of 1024 rows, 2048 -> 7168: 285 us (3.4) and 215 us (4.5; 238 with one copy per row instead of boxes of 32 x 64).  Under back-to-back calls the power limit takes a third of that.
// What bounds it is the work in shared memory: a K-block brings 32 KiB per CTA by TMA, the MMAs read as much, and the nvfp4 scales
// are written, transposed and copied on, 24 KiB more; half of that for mxfp4, which is what it is faster by.
// Tried in place of this arrangement (nvfp4 / mxfp4 us for the first of these sizes, 240 / 184 as it is):
//   two sets of scale warps that take groups in turn               248 / 188   the copies' latency is hidden already
//   stages of two K-blocks, half as many barrier turns             237 / 213   less lookahead
//   scales stored to tensor memory from registers, no transpose    268 / 217   four warps, one per lane quarter, read every word
//
// Barriers: as in grouped_gemm_mx2.cu, bar_sf counts the three scale warps of each CTA;
// bar_sfe[group], in each CTA, tells that tensor memory has the scales of the group's K-blocks.
#include "../common/fp4.cuh"
#include "expert_gemm.cuh"

namespace cam {

constexpr int kF4Threads = 768;
constexpr int kF4EpiThreads = 512;
constexpr int kF4SfWarp0 = 4, kF4EpiWarp0 = 8;
constexpr int kF4K = 256;                      // values of one K-block
constexpr int kF4Tile = 128 * 128;             // 128 rows of one K-block, 16 KiB
constexpr int kF4StageBytes = 2 * kF4Tile;
constexpr int kF4SfBlock = 4 * 512;            // scales of 128 rows (mxfp4 uses half)
constexpr int kF4SfStage = 3 * kF4SfBlock;
constexpr int kF4SfGroup = 4;                  // K-blocks whose scales travel together
constexpr int kF4SfSlots = 2 * kF4SfGroup;     // two groups
constexpr int kF4StgBox = 32 * 128;             // 32 bf16 rows of 64 columns
constexpr int kF4StgBytes = 8 * kF4StgBox;
// the plain form gives up a stage for the staging of its rows
__host__ __device__ constexpr int fp4_stages(bool swiglu) { return swiglu ? 5 : 4; }
__host__ __device__ constexpr int fp4_smem(bool swiglu) {
    return fp4_stages(swiglu) * kF4StageBytes + kF4SfSlots * kF4SfStage + (swiglu ? 0 : kF4StgBytes) + 1024;
}
static_assert(fp4_smem(true) <= 232448 && fp4_smem(false) <= 232448, "exceeds the shared memory of one CTA");
constexpr uint32_t kF4TmemCols = 512, kF4SfCol0 = 256, kF4SfCols = 48;
static_assert(kF4SfCol0 + fp4_stages(true) * kF4SfCols <= kF4TmemCols, "tensor memory");
// setmaxnreg: the shares must not exceed what the CTA was launched with (checked against ptxas by the build)
constexpr uint32_t kF4LaunchRegs = 80, kF4CtrlRegs = 32, kF4SfRegs = 56, kF4EpiRegs = 96;
static_assert(128 * kF4CtrlRegs + 128 * kF4SfRegs + kF4EpiThreads * kF4EpiRegs <= kF4LaunchRegs * kF4Threads,
              "setmaxnreg budget exceeds the registers the CTA owns: the kernel would hang");

namespace {

// D (+)= (A sfa) (B sfb), e2m1 x e2m1, on the pair; the formats differ in the scales' type and block
template <int FMT>
__device__ __forceinline__ void tc_mma_fp4_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                                uint32_t accumulate, uint32_t sfa_tmem, uint32_t sfb_tmem) {
    if constexpr (FMT == kFp4Nv) {
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n"
            "}\n" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(sfa_tmem), "r"(sfb_tmem)
            : "memory");
    } else {
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n"
            "}\n" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(sfa_tmem), "r"(sfb_tmem)
            : "memory");
    }
}

// 32 rows x 16 bytes of shared memory to 32 lanes x 4 columns of tensor memory, repeated in all four lane quarters, in both CTAs
__device__ __forceinline__ void tc_copy_scales_pair(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

}  // namespace

template <int FMT, bool SWIGLU>
__global__ void __launch_bounds__(kF4Threads, 1)
grouped_gemm_fp4_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_a32,
                        const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ CUtensorMap tmap_out, const GroupedGemmFp4Params p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {  // swizzled TMA tiles need it; the same in both CTAs of a pair
        if (threadIdx.x == 0) record_status(p.status, CAM_ERR_BAD_INDEX, 4, static_cast<int>(smem_u32(smem) & 1023u));
        return;
    }
    constexpr int NS = fp4_stages(SWIGLU);
    constexpr int SFW = FMT == kFp4Nv ? 4 : 2;  // scale words of a row and K-block
    constexpr int BLK = fp4_block(FMT);
    uint8_t* sfm = smem + NS * kF4StageBytes;
    uint8_t* stg = sfm + kF4SfSlots * kF4SfStage;
    uint8_t* ctrl = stg + (SWIGLU ? 0 : kF4StgBytes);
    uint64_t* bar_full = reinterpret_cast<uint64_t*>(ctrl);  // first CTA: TMA bytes of both CTAs' stage have landed
    uint64_t* bar_sf = bar_full + NS;                        // first CTA: a group of scale slots of both CTAs is ready
    uint64_t* bar_sfe = bar_sf + 2;                          // each CTA: a group of scale slots has been copied to tensor memory
    uint64_t* bar_empty = bar_sfe + 2;                       // each CTA: the MMAs that read a stage have retired
    uint64_t* bar_tfull = bar_empty + NS;                    // each CTA: accumulator of a tile is complete
    uint64_t* bar_tempty = bar_tfull + 1;                    // first CTA: both accumulators have been drained
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_tempty + 1);
    volatile uint32_t* abort_flag = tmem_slot + 1;

    const int warp = static_cast<int>(threadIdx.x) >> 5;
    const uint32_t lane = lane_id();
    const uint32_t cta = cluster_cta_rank();  // 0 = first CTA of the pair (issues the MMAs)
    const int pair_id = static_cast<int>(blockIdx.x) >> 1;
    const int num_pairs = static_cast<int>(gridDim.x) >> 1;
    const int kblocks = (p.k_dim + kF4K - 1) / kF4K;
    const int half_n = p.n_dim / 2;
    const int n_tiles = SWIGLU ? half_n / 128 : (p.n_dim + 255) / 256;

    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&bar_full[s], 1);
            mbar_init(&bar_empty[s], 1);
        }
        for (int j = 0; j < 2; ++j) {
            mbar_init(&bar_sf[j], 6);
            mbar_init(&bar_sfe[j], 1);
        }
        mbar_init(bar_tfull, 1);
        mbar_init(bar_tempty, 2 * (kF4EpiThreads / 32));
        *abort_flag = 0u;
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, kF4TmemCols);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();  // both CTAs' barriers are initialised before anything signals them
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    pdl_wait();
    pdl_release();
    PairTileWalker w(p.expert_offsets, p.num_experts, n_tiles, p.rows);
    int e, nt, row0, rows;
    bool ok = true;
    // first weight row of the lower / upper half of a tile
    auto b_row = [&](int half) { return e * p.n_dim + (SWIGLU ? half * half_n + nt * 128 : nt * 256 + half * 128); };

    if (warp < kF4SfWarp0) {
        reg_dealloc<kF4CtrlRegs>();
        const uint32_t abort_at = smem_u32(tmem_slot + 1);
        const uint32_t full_at = smem_u32(bar_full), sf_at = smem_u32(bar_sf), sfe_at = smem_u32(bar_sfe), empty_at = smem_u32(bar_empty);
        if (warp == 0) {
            // ------------------------------------------------------------ TMA producer (both CTAs)
            const bool leader = elect_one();
            if (leader) {
                prefetch_tensormap(&tmap_a);
                prefetch_tensormap(&tmap_a32);
                prefetch_tensormap(&tmap_b);
            }
            Ring ring;
            uint32_t ready = 1u;  // the first turn of every stage is free
            const uint32_t full0 = map_to_cta(bar_full, 0);
            // Only 32-row pieces of A that hold rows are loaded; what stays in the other rows of the stage reaches
            // accumulator rows that nobody reads.
            auto pieces = [](int r) { return r > 96 ? 4 : r > 0 ? (r + 31) / 32 : 0; };
            for (int tile = pair_id; !aborted(abort_flag) && w.locate(tile, e, nt, row0, rows); tile += num_pairs) {
                const int p0 = pieces(min(rows, BM)), p1 = pieces(rows - BM);
                const int mine = cta ? p1 : p0;
                const uint32_t bytes = 2u * kF4Tile + static_cast<uint32_t>(p0 + p1) * 4096u;
                const int arow = row0 + static_cast<int>(cta) * BM, brow = b_row(static_cast<int>(cta));
                for (int kb = 0; kb < kblocks; ++kb) {
                    const uint32_t s = ring.s;
                    if (!ready) mbar_wait_warp(empty_at + 8u * s, ring.ph ^ 1u, abort_at);
                    ring.next(NS);
                    ready = mbar_test(empty_at + 8u * ring.s, ring.ph ^ 1u);
                    if (leader) {
                        uint8_t* sa = smem + s * kF4StageBytes;
                        const uint32_t bar = full0 + 8u * s;
                        if (cta == 0) mbar_arrive_expect_tx(&bar_full[s], bytes);
                        tma_load_2d_pair(sa + kF4Tile, &tmap_b, bar, kb * 128, brow);
                        if (mine == 4) tma_load_2d_pair(sa, &tmap_a, bar, kb * 128, arow);
                        else for (int i = 0; i < mine; ++i) tma_load_2d_pair(sa + i * 4096, &tmap_a32, bar, kb * 128, arow + i * 32);
                    }
                    __syncwarp();
                }
            }
            if (leader && *abort_flag) record_status(p.status, CAM_ERR_TIMEOUT_PIPELINE, 0, 0);
        } else if (warp == 1 && cta == 0) {
            // ------------------------------------------------------------ MMA issuer (first CTA only)
            const bool leader = elect_one();
            Ring ring, groups;
            uint32_t tcount = 0, ready = 0u;
            for (int tile = pair_id; !aborted(abort_flag) && w.locate(tile, e, nt, row0, rows); tile += num_pairs, ++tcount) {
                // both epilogues must have drained the previous tile before its columns are overwritten
                mbar_wait_warp(smem_u32(bar_tempty), (tcount & 1u) ^ 1u, abort_at);
                tc_fence_after_sync();
                for (int kb = 0; kb < kblocks; ++kb) {
                    const uint32_t s = ring.s, gr = groups.s, in_group = static_cast<uint32_t>(kb) % kF4SfGroup;
                    const bool group_ends = in_group == kF4SfGroup - 1 || kb == kblocks - 1;
                    if (in_group == 0) mbar_wait_warp(sf_at + 8u * gr, groups.ph, abort_at);
                    if (!ready) mbar_wait_warp(full_at + 8u * s, ring.ph, abort_at);
                    tc_fence_after_sync();
                    ring.next(NS);
                    if (group_ends) groups.next(2);
                    ready = mbar_test(full_at + 8u * ring.s, ring.ph);
                    const uint32_t sa = smem_u32(smem) + s * kF4StageBytes;
                    const uint64_t adesc = umma_desc_k_sw128(sa), bdesc = umma_desc_k_sw128(sa + kF4Tile);
                    const uint32_t sfs = smem_u32(sfm) + (gr * kF4SfGroup + in_group) * kF4SfStage;
                    const uint32_t sf = tmem_base + kF4SfCol0 + s * kF4SfCols;  // SFW x (4 columns of A, 8 of B)
                    if (leader) {
#pragma unroll
                        for (int k = 0; k < SFW; ++k) {
                            tc_copy_scales_pair(sf + 12u * k, desc_scales(sfs + k * 512));
                            tc_copy_scales_pair(sf + 12u * k + 4u, desc_scales(sfs + kF4SfBlock + k * 512));
                            tc_copy_scales_pair(sf + 12u * k + 8u, desc_scales(sfs + 2 * kF4SfBlock + k * 512));
                        }
                        if (group_ends) tc_commit_both(sfe_at + 8u * gr);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {  // 64 values = 32 bytes (2 x 16) further along K inside the swizzle atom
                            const uint32_t c = sf + 12u * (FMT == kFp4Nv ? k : k >> 1);
                            tc_mma_fp4_pair<FMT>(tmem_base, adesc + 2u * k, bdesc + 2u * k,
                                                 idesc_fp4<FMT>(2 * BM, 256, FMT == kFp4Nv ? 0u : 2u * (k & 1)), (kb | k) ? 1u : 0u, c, c + 4u);
                        }
                        tc_commit_both(empty_at + 8u * s);  // the stage, in both CTAs, is reusable once these have retired
                    }
                    __syncwarp();
                }
                if (leader) tc_commit_both(smem_u32(bar_tfull));
                __syncwarp();
            }
            if (leader && *abort_flag) record_status(p.status, CAM_ERR_TIMEOUT_PIPELINE, 1, static_cast<int>(tcount));
        }
    } else if (warp < kF4EpiWarp0) {
        reg_dealloc<kF4SfRegs>();
        // ---------------------------------------------------------------- scale warps: rows, lower and upper weight rows
        const int what = warp - kF4SfWarp0;
        if (what < 3) {
            const int pitch = p.k_dim / BLK;          // bytes of scales of a row
            const int words = pitch / 4;
            const int last_b = p.num_experts * p.n_dim - 1;
            const int sub = static_cast<int>(lane) >> 2, piece = static_cast<int>(lane) & 3;  // row of 8, K-block of the group
            uint8_t* block = sfm + what * kF4SfBlock;
            Ring groups;
            for (int tile = pair_id; ok && w.locate(tile, e, nt, row0, rows); tile += num_pairs) {
                // Past the tile's rows nothing is loaded: those accumulator rows are not read.  (Loading some row there instead
                // made all SMs ask one L2 slice for the same bytes: 8 rows of 8 experts, 4096 x 7168, 231 us.)
                // A block of weight rows past the last one (its columns are not stored either) is left out.
                const int first = what == 0 ? row0 + static_cast<int>(cta) * BM : b_row(what - 1);
                const int live = what == 0 ? rows - static_cast<int>(cta) * BM : first < last_b ? 128 : 0;
                const uint8_t* from = (what == 0 ? p.a_scales : p.b_scales) + static_cast<size_t>(first + sub) * pitch + piece * (SFW * 4);
                for (int kb = 0; kb < kblocks; kb += kF4SfGroup, groups.next(2)) {
                    const bool got = mbar_wait_bounded(&bar_sfe[groups.s], groups.ph ^ 1u, abort_flag);
                    if (!__all_sync(0xFFFFFFFFu, got)) { ok = false; break; }
                    uint8_t* slots = block + groups.s * (kF4SfGroup * kF4SfStage);
                    const uint32_t dst = smem_u32(slots) + static_cast<uint32_t>(piece) * kF4SfStage + static_cast<uint32_t>(sub) * 16u;
                    const int left = words - (kb + piece) * SFW;  // words of the row that this lane's piece can have
                    if (p.scale_vec) {
                        if (left > 0) {
                            const uint8_t* at = from;
#pragma unroll
                            for (int i = 0; i < 16; ++i, at += 8 * pitch)  // rows 8 i + sub
                                if (8 * i + sub < live) copy_async<SFW * 4>(dst + fp4_scale_at<FMT>(i >> 2) + (i & 3) * 128u, at, true);
                        }
                    } else {
                        for (int i = 0; i < 16; ++i) {
                            if (8 * i + sub >= live) break;
                            const uint8_t* at = from + static_cast<size_t>(8 * i) * pitch;
#pragma unroll
                            for (int j = 0; j < SFW; ++j)
                                copy_async<4>(dst + fp4_scale_at<FMT>(i >> 2) + (i & 3) * 128u + j * 4u, j < left ? at + j * 4 : p.a_scales, j < left);
                        }
                    }
                    from += kF4SfGroup * SFW * 4;
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    __syncwarp();  // the words a lane transposes were copied by others
#pragma unroll
                    for (int c = 0; c < kF4SfGroup; ++c) fp4_transpose_scales<FMT>(slots + c * kF4SfStage + lane * 16u);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {  // the first CTA's barrier counts the warps of both CTAs
                        if (cta == 0) mbar_arrive(&bar_sf[groups.s]);
                        else mbar_arrive_cluster(map_to_cta(&bar_sf[groups.s], 0));
                    }
                }
            }
            if (!ok && lane == 0) record_status(p.status, CAM_ERR_TIMEOUT_PIPELINE, 3, static_cast<int>(groups.s));
        }
    } else {
        reg_alloc<kF4EpiRegs>();
        // ---------------------------------------------------------------- epilogue warps
        const int ew = warp - kF4EpiWarp0;
        const int q = warp & 3;   // TMEM lane quarter this warp may read
        const int cq = ew >> 2;   // which 32-column quarter of each 128-column half
        const int r = q * 32 + static_cast<int>(lane);
        const float a_g = p.a_gscale != nullptr ? __ldg(p.a_gscale) : 1.f;
        const float out_g = p.out_gscale != nullptr ? __ldg(p.out_gscale) : 1.f;
        uint32_t tcount = 0;
        for (int tile = pair_id; w.locate(tile, e, nt, row0, rows); tile += num_pairs, ++tcount) {
            row0 += static_cast<int>(cta) * BM;
            rows = max(0, min(BM, rows - static_cast<int>(cta) * BM));
            const bool valid = r < rows;
            const size_t grow = static_cast<size_t>(row0 + (valid ? r : 0));
            const float alpha = p.b_gscale != nullptr ? a_g * __ldg(p.b_gscale + e) : a_g;
            epilogue_wait(bar_tfull, tcount & 1u, abort_flag, 64u);
            tc_fence_after_sync();
            const uint32_t t0 = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + cq * 32;
            uint32_t v0[32], v1[32];  // columns cq*32.. of the first 128-column half, same of the second
            tmem_ld_32x32b_x32(t0, v0);
            tmem_ld_32x32b_x32(t0 + 128, v1);
            tc_wait_ld_regs(v0);
            tc_wait_ld_regs(v1);
            // the tile now lives in registers: hand the accumulator back to the MMA issuer
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if (cta == 0) mbar_arrive(bar_tempty);
                else mbar_arrive_cluster(map_to_cta(bar_tempty, 0));
            }
            if constexpr (SWIGLU) {
                uint4 codes;
                uint32_t scales;
                fp4_swiglu32<FMT>(v0, v1, alpha, out_g, codes, scales);
                if (valid) {
                    const size_t at = grow * (half_n / 32) + nt * 4 + cq;  // in units of 32 columns
                    *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + at * 16) = codes;
                    if (FMT == kFp4Nv) *reinterpret_cast<uint16_t*>(p.out_scales + at * 2) = static_cast<uint16_t>(scales);
                    else p.out_scales[at] = static_cast<uint8_t>(scales);
                }
            } else {
                // Two warps share 32 rows x 64 columns, which go through shared memory as bf16 and leave as one tensor copy; rows of a
                // block of 32 that ends inside it are stored from registers.
                const int box = q * 2 + (cq >> 1);
                uint8_t* at = stg + box * kF4StgBox + lane * 128;
                const bool whole = rows >= q * 32 + 32, issues = (cq & 1) == 0 && lane == 0;
                auto push_half = [&](const uint32_t (&v)[32], int c0) {
                    uint4 o[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        o[j] = pack_bf16x8(__uint_as_float(v[8 * j]) * alpha, __uint_as_float(v[8 * j + 1]) * alpha, __uint_as_float(v[8 * j + 2]) * alpha,
                                           __uint_as_float(v[8 * j + 3]) * alpha, __uint_as_float(v[8 * j + 4]) * alpha, __uint_as_float(v[8 * j + 5]) * alpha,
                                           __uint_as_float(v[8 * j + 6]) * alpha, __uint_as_float(v[8 * j + 7]) * alpha);
                    if (whole) {  // the same in both warps
                        if (issues) bulk_wait_group_read<0>();  // the copy that reads this buffer is done with it
                        named_bar_sync(1 + box, 64);
#pragma unroll
                        for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(at + ((((cq & 1) * 4 + j) ^ (static_cast<int>(lane) & 7)) << 4)) = o[j];
                        fence_proxy_async_smem();
                        named_bar_sync(1 + box, 64);
                        if (issues) {
                            tma_store_2d(&tmap_out, smem_u32(stg + box * kF4StgBox), (c0 + (cq >> 1) * 64) * 2, row0 + q * 32);
                            bulk_commit_group();
                        }
                    } else if (valid) {
                        uint4* to = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + grow * p.n_dim + c0 + cq * 32);
#pragma unroll
                        for (int j = 0; j < 4; ++j) to[j] = o[j];
                    }
                };
                const int c_lo = nt * 256;
                push_half(v0, c_lo);
                if (c_lo + 128 < p.n_dim) push_half(v1, c_lo + 128);  // same answer in every thread of the CTA
            }
        }
        if (!SWIGLU && (cq & 1) == 0) bulk_wait_group<0>();  // everything this thread sent has been written
        if (*abort_flag) record_status(p.status, CAM_ERR_TIMEOUT_PIPELINE, 2, static_cast<int>(tcount));
        // rows of no expert
        const int et = static_cast<int>(threadIdx.x) - kF4EpiWarp0 * 32;
        if constexpr (SWIGLU) {
            zero_loose_rows(p.out, half_n / 32, p.expert_offsets, p.num_experts, p.rows, et, kF4EpiThreads);
            zero_loose_scales(p.out_scales, half_n / BLK, p.expert_offsets, p.num_experts, p.rows, et, kF4EpiThreads);
        } else {
            zero_loose_rows(p.out, p.n_dim / 8, p.expert_offsets, p.num_experts, p.rows, et, kF4EpiThreads);
        }
    }

    // ------------------------------------------------------------------ teardown
    abort_drain(abort_flag);
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();  // the other CTA may still read this CTA's shared memory or signal its barriers
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem_base, kF4TmemCols);
    }
}

}  // namespace cam

namespace {

template <int FMT, bool SWIGLU>
int launch_fp4(const cam::GroupedGemmFp4Params* p, const CUtensorMap* ta, const CUtensorMap* ta32, const CUtensorMap* tb, const CUtensorMap* tout, cudaStream_t stream) {
    static cam::PairLimit limit;
    // at most one row block per expert beyond the full ones
    const int64_t n_tiles = SWIGLU ? p->n_dim / 256 : (p->n_dim + 255) / 256;
    const int64_t blocks = p->rows / 256 + (p->rows < p->num_experts ? p->rows : p->num_experts);
    return cam::launch_pairs(limit, cam::grouped_gemm_fp4_kernel<FMT, SWIGLU>, cam::kF4Threads, cam::fp4_smem(SWIGLU), blocks * n_tiles, stream, *ta, *ta32, *tb, *tout, *p);
}

}  // namespace

extern "C" int cam_launch_grouped_gemm_fp4(const cam::GroupedGemmFp4Params* p, int fmt, int swiglu, const CUtensorMap* tmap_a,
                                           const CUtensorMap* tmap_a32, const CUtensorMap* tmap_b, const CUtensorMap* tmap_out, cudaStream_t stream) {
    if (fmt == cam::kFp4Nv)
        return swiglu ? launch_fp4<cam::kFp4Nv, true>(p, tmap_a, tmap_a32, tmap_b, tmap_out, stream) : launch_fp4<cam::kFp4Nv, false>(p, tmap_a, tmap_a32, tmap_b, tmap_out, stream);
    return swiglu ? launch_fp4<cam::kFp4Mx, true>(p, tmap_a, tmap_a32, tmap_b, tmap_out, stream) : launch_fp4<cam::kFp4Mx, false>(p, tmap_a, tmap_a32, tmap_b, tmap_out, stream);
}
