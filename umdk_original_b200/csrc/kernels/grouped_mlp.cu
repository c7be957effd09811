// Gated feed-forward block of 16-bit experts, forward and backward, on CTA pairs with fp32 accumulators.  For the rows r of
// expert e (w1 [E, 2I, h] with the gate rows first, w2 [E, h, I]):
//   up      g = x Wg^T, u = x Wu^T, act = silu(g) u            one kernel: both projections, the activation, the product
//   down    y = act W2^T
//   dact    da = dy W2, s = 1 / (1 + e^-g):  dg = da u s (1 + g (1 - s)),  du = da g s    one kernel, da never leaves it
//   dx      dx = dg Wg + du Wu = dgu W1
//   dw      dW2 = dy^T act,  dW1 = dgu^T x, the sums over the rows of the expert
// What is rounded to 16 bits: act and dgu, because they are operands of the next product and the tensor core takes no wider ones at
// this rate, and the results.  Gate and up are kept in fp32 for the backward pass and da stays in the accumulator, so that no result is
// more than one rounding of an operand and its own away from the formula: the relative error of y, dx and both weight gradients is
// 1.41 times what it would be with act and dgu in fp32 (256 rows, 1024 x 512: 2.34e-3 against 1.66e-3 in bf16, 2.93e-4 against
// 2.07e-4 in fp16).  In fp16 it is also a limit of range: act and dgu past 65504 become infinite where the formula's result might not.
//
// up, down and dx (grouped_gemm_16_rows_kernel): the weights are the M operand of the tensor core, the rows of the expert its N
// operand in steps of 32, so that the tensor time, and at the power limit the energy, follow the rows present: an expert of 375
// rows is two tiles of 192, where tiles of 256 rows as M operand compute 512.  A pair of CTAs computes 512 weight rows (each CTA two
// blocks of 128: the gate and the up block of the same features, or neighbouring blocks) x up to 256 rows, of which each CTA loads
// half; a K-block of 64 values brings 96 KiB to the pair for 1024 cycles of MMAs, three quarters of what tiles of 256 x 256 need.
// The accumulators fill tensor memory, so the epilogue takes them to registers at once, rounded, and hands them back before it
// stores.  Against 256 x 256 tiles in a steady loop: 24 uneven experts of 375 rows, 4096 x 1024 294 -> 278 us, 16 of 375 rows, 4096
// x 2048 370 -> 337, 8 of 512 rows, 7168 x 2048 397 -> 378.
//
// dact and dw (grouped_gemm_16_square_kernel): tiles of 256 x 256 and two accumulators in turn.  dact reads 8 bytes of gate and up
// for every value of da, and its epilogue is what takes long: with an accumulator to spare it runs beside the MMAs of the next tile
// (16 x 1024 rows, 4096 x 2048: 225 us, with 512 x 256 tiles 288).
// The weight gradients are written by tensor copies of 64 columns x 128 rows, one instruction each, from two buffers that half of the
// epilogue fills on its own: 16 gradients of 4096 x 2048 from 16 rows each (268 MB) 104 -> 52 us against one copy per row, 0.8 of a
// plain copy's rate, and 512 rows 125 -> 102.
//
// The other products write boxes of 32 rows x 64 columns, each filled by two warps; the last, ragged rows of a block are stored from
// registers.  Against one copy per row: up and down of 4 experts of 7168 x 2048, 256 rows 123 -> 116 us, dact and dx 115 -> 109.
//
// With few rows per expert, or few tiles in all, up, down, dact and dx are computed by expert_gemm_narrow.cu instead.
//
// K-blocks of 64 values (128 bytes) come by TMA.  An operand whose contraction index is not its contiguous one (w2 of dact, w1 of dx,
// both operands of dw) is loaded as [64 of the contraction][64 values] boxes and read by the tensor core in its MN-major form;
// nothing is transposed in memory.
//
// The sum of dw runs over a ragged number of rows.  The last K-block of an expert then holds rows of the next one: its loads
// complete on a barrier of their own, a warp overwrites those rows with zeros in shared memory (in both operands: a NaN times
// zero would stay) and only then raises the stage's barrier.
#include "expert_gemm.cuh"

namespace cam {

constexpr int kEmThreads = 640;
constexpr int kEmEpiThreads = 512;
constexpr int kEmEpiWarp0 = 4;
constexpr int kEmStages = 6;
constexpr int kEmTile = 128 * 128;  // 128 rows x 64 values of A, or as many of B
constexpr int kEmStageBytes = 2 * kEmTile;
constexpr int kEmStgBytes = 32768;  // results on their way out: 128 rows x 128 columns of 16 bits, in boxes 128 bytes wide
constexpr int kEmSmem = kEmStages * kEmStageBytes + kEmStgBytes + 1024;
static_assert(kEmSmem <= 232448, "exceeds the shared memory of one CTA");
constexpr uint32_t kEmTmemCols = 512;
// setmaxnreg: the shares must not exceed what the CTA was launched with (checked against ptxas by the build)
constexpr uint32_t kEmLaunchRegs = 96, kEmCtrlRegs = 40, kEmEpiRegs = 104;
static_assert(128 * kEmCtrlRegs + kEmEpiThreads * kEmEpiRegs <= kEmLaunchRegs * kEmThreads,
              "setmaxnreg budget exceeds the registers the CTA owns: the kernel would hang");

namespace {

__device__ __forceinline__ void tc_mma_16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const void* tmap, uint32_t bar_cluster_addr, int32_t c0, int32_t c1, int32_t c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar_cluster_addr), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

// Tiles of the weight gradients: 256 x 256 of every expert's [m_dim, n_dim]; `rows` are the rows summed over.
struct GradTileWalker {
    const int* off;
    int num_experts, m_tiles, n_tiles, rows_total;
    __device__ GradTileWalker(const int* o, int ne, int mt, int nt, int rt) : off(o), num_experts(ne), m_tiles(mt), n_tiles(nt), rows_total(rt) {}
    __device__ bool locate(int tile, int& e, int& mt, int& nt, int& row0, int& rows) const {
        const int per = m_tiles * n_tiles;
        e = tile / per;
        if (e >= num_experts) return false;
        const int local = tile - e * per;
        mt = local / n_tiles;
        nt = local - mt * n_tiles;
        row0 = expert_bound(off, e, rows_total);
        rows = max(expert_bound(off, e + 1, rows_total) - row0, 0);
        return true;
    }
};

}  // namespace

// Tiles of 256 x 256 with two accumulators in turn.  DW: weight gradients (contraction over an expert's rows, both operands
// MN-major).  Otherwise dact: 256 rows x 256 columns of da, the weights MN-major.
template <bool DW>
__global__ void __launch_bounds__(kEmThreads, 1)
grouped_gemm_16_square_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_a32,
                       const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ CUtensorMap tmap_out, const GroupedMlpParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {  // swizzled TMA tiles need it; the same in both CTAs of a pair
        if (threadIdx.x == 0) record_status(p.status, CAM_ERR_BAD_INDEX, 4, static_cast<int>(smem_u32(smem) & 1023u));
        return;
    }
    constexpr int NS = kEmStages;
    uint8_t* stg = smem + NS * kEmStageBytes;
    uint8_t* ctrl = stg + kEmStgBytes;
    uint64_t* bar_full = reinterpret_cast<uint64_t*>(ctrl);  // first CTA: bytes of both CTAs' stage have landed
    uint64_t* bar_empty = bar_full + NS;                     // each CTA: the MMAs that read a stage have retired
    uint64_t* bar_tfull = bar_empty + NS;                    // each CTA, [2]: accumulator of a tile is complete
    uint64_t* bar_tempty = bar_tfull + 2;                    // first CTA, [2]: both CTAs have drained the accumulator
    uint64_t* bar_tail = bar_tempty + 2;                     // each CTA, per stage: its bytes of a ragged last K-block have landed
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_tail + NS);
    volatile uint32_t* abort_flag = tmem_slot + 1;

    const int warp = static_cast<int>(threadIdx.x) >> 5;
    const uint32_t lane = lane_id();
    const uint32_t cta = cluster_cta_rank();  // 0 = first CTA of the pair (issues the MMAs)
    const int pair_id = static_cast<int>(blockIdx.x) >> 1;
    const int num_pairs = static_cast<int>(gridDim.x) >> 1;
    const int n_tiles = (p.n_dim + 255) / 256;

    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&bar_full[s], DW ? 2 : 1);
            mbar_init(&bar_empty[s], 1);
            mbar_init(&bar_tail[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bar_tfull[b], 1);
            mbar_init(&bar_tempty[b], 2 * (kEmEpiThreads / 32));
        }
        *abort_flag = 0u;
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, kEmTmemCols);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();  // both CTAs' barriers are initialised before anything signals them
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    pdl_wait();
    pdl_release();
    PairTileWalker wr(p.expert_offsets, p.num_experts, n_tiles, p.rows);
    const GradTileWalker wg(p.expert_offsets, p.num_experts, (p.m_dim + 255) / 256, n_tiles, p.rows);
    int e, mt = 0, nt, row0, rows;
    bool ok = true;
    auto locate = [&](int tile) { return DW ? wg.locate(tile, e, mt, nt, row0, rows) : wr.locate(tile, e, nt, row0, rows); };
    auto kblocks_of = [&]() { return ((DW ? rows : p.k_dim) + 63) / 64; };

    if (warp < kEmEpiWarp0) {
        reg_dealloc<kEmCtrlRegs>();
        const uint32_t abort_at = smem_u32(tmem_slot + 1);
        const uint32_t full_at = smem_u32(bar_full), empty_at = smem_u32(bar_empty);
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
            const uint32_t full0 = map_to_cta(bar_full, 0), tail_own = map_to_cta(bar_tail, cta);
            // dact: only 32-row pieces of A that hold rows are loaded; what stays in the other rows of the stage reaches
            // accumulator rows that nobody reads
            auto pieces = [](int r) { return r > 96 ? 4 : r > 0 ? (r + 31) / 32 : 0; };
            for (int tile = pair_id; !aborted(abort_flag) && locate(tile); tile += num_pairs) {
                const int kblocks = kblocks_of();
                const int p0 = pieces(min(rows, BM)), p1 = pieces(rows - BM), mine = cta ? p1 : p0;
                const uint32_t bytes = DW ? 2u * kEmStageBytes : 2u * kEmTile + static_cast<uint32_t>(p0 + p1) * 4096u;
                const int half = static_cast<int>(cta);
                for (int kb = 0; kb < kblocks; ++kb) {
                    const uint32_t s = ring.s;
                    if (!ready) mbar_wait_warp(empty_at + 8u * s, ring.ph ^ 1u, abort_at);
                    ring.next(NS);
                    ready = mbar_test(empty_at + 8u * ring.s, ring.ph ^ 1u);
                    if (leader) {
                        uint8_t* sa = smem + s * kEmStageBytes;
                        uint8_t* sb = sa + kEmTile;
                        uint32_t bar = full0 + 8u * s;
                        if (DW && kb == kblocks - 1 && (rows & 63) != 0) {
                            bar = tail_own + 8u * s;
                            mbar_arrive_expect_tx(&bar_tail[s], kEmStageBytes);
                        } else if (cta == 0) {
                            mbar_arrive_expect_tx(&bar_full[s], bytes);
                        } else if (DW) {
                            mbar_arrive_cluster(bar);
                        }
                        if constexpr (DW) {
                            const int r = row0 + kb * 64, ca = (mt * 256 + half * 128) * 2, cb = (nt * 256 + half * 128) * 2;
                            tma_load_2d_pair(sa, &tmap_a, bar, ca, r);
                            tma_load_2d_pair(sa + 8192, &tmap_a, bar, ca + 128, r);
                            tma_load_2d_pair(sb, &tmap_b, bar, cb, r);
                            tma_load_2d_pair(sb + 8192, &tmap_b, bar, cb + 128, r);
                        } else {
                            const int cb = (nt * 256 + half * 128) * 2;
                            tma_load_3d_pair(sb, &tmap_b, bar, cb, kb * 64, e);
                            tma_load_3d_pair(sb + 8192, &tmap_b, bar, cb + 128, kb * 64, e);
                            const int arow = row0 + half * BM;
                            if (mine == 4) tma_load_2d_pair(sa, &tmap_a, bar, kb * 128, arow);
                            else for (int i = 0; i < mine; ++i) tma_load_2d_pair(sa + i * 4096, &tmap_a32, bar, kb * 128, arow + i * 32);
                        }
                    }
                    __syncwarp();
                }
            }
            if (leader && *abort_flag) record_status(p.status, CAM_ERR_TIMEOUT_PIPELINE, 0, 0);
        } else if (warp == 1 && cta == 0) {
            // ------------------------------------------------------------ MMA issuer (first CTA only)
            const bool leader = elect_one();
            // fp32 accumulator; a_major / b_major (bits 15, 16) = 1 for MN-major operands
            const uint32_t idesc = umma_idesc(2 * BM, 256, 1u, p.fp16 ? 0u : 1u) | (DW ? 1u << 15 : 0u) | (1u << 16);
            Ring ring;
            uint32_t tcount = 0, ready = 0u;
            for (int tile = pair_id; !aborted(abort_flag) && locate(tile); tile += num_pairs, ++tcount) {
                const int kblocks = kblocks_of();
                const uint32_t b = tcount & 1u;
                // both epilogues must have drained this accumulator's previous tile
                mbar_wait_warp(smem_u32(&bar_tempty[b]), ((tcount >> 1) & 1u) ^ 1u, abort_at);
                tc_fence_after_sync();
                for (int kb = 0; kb < kblocks; ++kb) {
                    const uint32_t s = ring.s;
                    if (!ready) mbar_wait_warp(full_at + 8u * s, ring.ph, abort_at);
                    tc_fence_after_sync();
                    ring.next(NS);
                    ready = mbar_test(full_at + 8u * ring.s, ring.ph);
                    const uint32_t sa = smem_u32(smem) + s * kEmStageBytes;
                    const uint64_t adesc = DW ? umma_desc_mn_sw128(sa) : umma_desc_k_sw128(sa);
                    const uint64_t bdesc = umma_desc_mn_sw128(sa + kEmTile);
                    if (leader) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)  // 16 of the contraction: 32 bytes of a row, or 16 rows of 128 bytes
                            tc_mma_16_pair(tmem_base + b * 256u, adesc + (DW ? 128u : 2u) * k, bdesc + 128u * k, idesc, (kb | k) ? 1u : 0u);
                        tc_commit_both(empty_at + 8u * s);
                    }
                    __syncwarp();
                }
                if (leader) tc_commit_both(smem_u32(&bar_tfull[b]));
                __syncwarp();
            }
            if (leader && *abort_flag) record_status(p.status, CAM_ERR_TIMEOUT_PIPELINE, 1, static_cast<int>(tcount));
        } else if (DW && warp == 2) {
            // ------------------------------------------------------------ zeros behind the last row (both CTAs)
            uint32_t it = 0, phases = 0;  // bit s: parity of stage s's next ragged block
            for (int tile = pair_id; ok && locate(tile); tile += num_pairs) {
                it += static_cast<uint32_t>(kblocks_of());
                const int live = rows & 63;
                if (live == 0) continue;
                const uint32_t s = (it - 1u) % NS;
                const bool got = mbar_wait_bounded(&bar_tail[s], (phases >> s) & 1u, abort_flag);
                if (!__all_sync(0xFFFFFFFFu, got)) { ok = false; break; }
                phases ^= 1u << s;
                uint8_t* at = smem + s * kEmStageBytes + live * 128;  // the swizzle moves bytes inside a 128-byte row only
                const int units = (64 - live) * 8;
                for (int c = 0; c < 4; ++c)
                    for (int i = static_cast<int>(lane); i < units; i += 32) *reinterpret_cast<uint4*>(at + c * 8192 + i * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (cta == 0) mbar_arrive(&bar_full[s]);
                    else mbar_arrive_cluster(map_to_cta(&bar_full[s], 0));
                }
            }
            if (!ok && lane == 0) record_status(p.status, CAM_ERR_TIMEOUT_PIPELINE, 5, static_cast<int>(it));
        }
    } else {
        reg_alloc<kEmEpiRegs>();
        // ---------------------------------------------------------------- epilogue warps
        const int ew = warp - kEmEpiWarp0;
        const int q = warp & 3;   // TMEM lane quarter this warp may read
        const int cq = ew >> 2;   // which 32-column quarter of each 128-column half
        const int r = q * 32 + static_cast<int>(lane);
        const bool fp16 = p.fp16 != 0;
        uint32_t tcount = 0;
        for (int tile = pair_id; locate(tile); tile += num_pairs, ++tcount) {
            const uint32_t b = tcount & 1u;
            const int first = (DW ? mt * 256 : 0) + static_cast<int>(cta) * BM;  // of this CTA's rows of the tile
            const bool valid = first + r < (DW ? p.m_dim : rows);
            const size_t orow_i = DW ? static_cast<size_t>(e) * p.m_dim + first + r : static_cast<size_t>(row0 + first + r);
            const bool empty = DW && rows == 0;
            const uint32_t t0 = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + b * 256u + cq * 32;
            auto hand_back = [&]() {  // what this warp needs of the accumulator is in registers
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if (cta == 0) mbar_arrive(&bar_tempty[b]);
                    else mbar_arrive_cluster(map_to_cta(&bar_tempty[b], 0));
                }
            };
            if constexpr (!DW) {
                // n_dim = I columns of da; dgu [rows, 2I].  16 columns at a time: their gate and up values are asked for before
                // the accumulator is waited for, or while the 16 before them are worked on.
                const float* gu0 = p.gate_up + orow_i * (2 * static_cast<size_t>(p.n_dim)) + nt * 256 + cq * 32;
                float g[16], u[16];
                auto load = [&](int part) {  // part 0..3: half part / 2, columns 16 (part % 2)
                    const int off = (part >> 1) * 128 + (part & 1) * 16;
#pragma unroll
                    for (int i = 0; i < 16; i += 8) {
                        if (valid && nt * 256 + cq * 32 + off + i < p.n_dim) {  // n_dim is a multiple of 8
                            ld_nc_f8(gu0 + off + i, g + i);
                            ld_nc_f8(gu0 + off + i + p.n_dim, u + i);
                        } else {
#pragma unroll
                            for (int j = 0; j < 8; ++j) g[i + j] = u[i + j] = 0.f;
                        }
                    }
                };
                load(0);
                epilogue_wait(&bar_tfull[b], (tcount >> 1) & 1u, abort_flag, 64u);
                tc_fence_after_sync();
                // Two warps share 32 rows x 64 columns, which go through shared memory and leave as one tensor copy; rows of a block of
                // 32 that ends inside it are stored from registers.  `part`: 0 dg, 1 du.
                const int box = q * 2 + (cq >> 1);
                uint8_t* at = stg + box * 4096 + lane * 128;
                const bool whole = first + q * 32 + 32 <= rows, issues = (cq & 1) == 0 && lane == 0;
                auto push = [&](const uint32_t* w16, int c0, int part) {
                    if (c0 + (cq >> 1) * 64 >= p.n_dim) return;  // the same in both warps
                    if (whole) {
                        if (issues) bulk_wait_group_read<0>();  // the copy that reads this buffer is done with it
                        named_bar_sync(1 + box, 64);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            *reinterpret_cast<uint4*>(at + ((((cq & 1) * 4 + j) ^ (r & 7)) << 4)) = make_uint4(w16[4 * j], w16[4 * j + 1], w16[4 * j + 2], w16[4 * j + 3]);
                        fence_proxy_async_smem();
                        named_bar_sync(1 + box, 64);
                        if (issues) {
                            tma_store_3d(&tmap_out, smem_u32(stg + box * 4096), (c0 + (cq >> 1) * 64) * 2, part, row0 + first + q * 32);
                            bulk_commit_group();
                        }
                    } else if (valid) {
                        const int c = c0 + cq * 32;
                        uint16_t* to = static_cast<uint16_t*>(p.out) + (2 * orow_i + part) * p.n_dim + c;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (c + 8 * j < p.n_dim) *reinterpret_cast<uint4*>(to + 8 * j) = make_uint4(w16[4 * j], w16[4 * j + 1], w16[4 * j + 2], w16[4 * j + 3]);
                    }
                };
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t v[32];
                    tmem_ld_32x32b_x32(t0 + h * 128, v);
                    tc_wait_ld_regs(v);
                    if (h == 1) hand_back();
                    const int c0 = nt * 256 + h * 128;
                    uint32_t du[16];
#pragma unroll
                    for (int part = 0; part < 2; ++part) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float a[4], d[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                gated_gradients(__uint_as_float(v[part * 16 + 4 * i + k]), g[4 * i + k], u[4 * i + k], a[k], d[k]);
                            }
                            v[part * 8 + 2 * i] = pack16(a[0], a[1], fp16);  // words 0..15: dg; their da has been used
                            v[part * 8 + 2 * i + 1] = pack16(a[2], a[3], fp16);
                            du[part * 8 + 2 * i] = pack16(d[0], d[1], fp16);
                            du[part * 8 + 2 * i + 1] = pack16(d[2], d[3], fp16);
                        }
                        if (2 * h + part < 3) load(2 * h + part + 1);
                    }
                    push(v, c0, 0);
                    push(du, c0, 1);
                }
                continue;
            }
            epilogue_wait(&bar_tfull[b], (tcount >> 1) & 1u, abort_flag, 64u);
            tc_fence_after_sync();
            uint32_t v0[32], v1[32];  // columns cq*32.. of the first 128-column half, same of the second
            tmem_ld_32x32b_x32(t0, v0);
            tmem_ld_32x32b_x32(t0 + 128, v1);
            tc_wait_ld_regs(v0);
            tc_wait_ld_regs(v1);
            hand_back();
            // 64 columns (two of the 32-column quarters, 8 warps) have a buffer of their own and leave as one copy
            const int pair = cq >> 1;
            uint8_t* row = stg + pair * 16384 + r * 128;
            const bool issues = (ew & 7) == 0 && lane == 0;  // the pair's first thread
            auto store_half = [&](uint32_t* v, int h) {
                const int c0 = nt * 256 + h * 128 + pair * 64;
                if (c0 >= p.n_dim) return;  // the same in every thread of the pair
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = empty ? 0u : pack16(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]), fp16);
                if (issues) bulk_wait_group_read<0>();  // the copy that reads this buffer is done with it
                named_bar_sync(1 + pair, kEmEpiThreads / 2);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    *reinterpret_cast<uint4*>(row + ((((cq & 1) * 4 + j) ^ (r & 7)) << 4)) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                fence_proxy_async_smem();
                named_bar_sync(1 + pair, kEmEpiThreads / 2);
                if (issues) {
                    if (first < p.m_dim) tma_store_3d(&tmap_out, smem_u32(stg + pair * 16384), c0 * 2, first, e);
                    bulk_commit_group();
                }
            };
            store_half(v0, 0);
            store_half(v1, 1);
        }
        if (DW ? (ew & 7) == 0 : (cq & 1) == 0) bulk_wait_group<0>();  // everything this thread sent has been written
        if (*abort_flag) record_status(p.status, CAM_ERR_TIMEOUT_PIPELINE, 2, static_cast<int>(tcount));
    }

    // ------------------------------------------------------------------ teardown
    abort_drain(abort_flag);
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();  // the other CTA may still read this CTA's shared memory or signal its barriers
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem_base, kEmTmemCols);
    }
}

// One CTA pair, rows as N operand.  W_MN: the weights' contraction index is their row index in memory.
constexpr int kErStages = 4;
constexpr int kErStageBytes = 3 * kEmTile;  // two blocks of 128 weight rows, half of the rows
constexpr int kErSmem = kErStages * kErStageBytes + kEmStgBytes + 1024;
static_assert(kErSmem <= 232448, "exceeds the shared memory of one CTA");

// Tiles of (expert, rows, weight rows): the rows of an expert in ceil(rows / 256) equal parts of whole 32s.
struct PartWalker {
    const int* off;
    int num_experts, n_tiles, rows_total;
    int e = 0, base = 0;
    __device__ PartWalker(const int* o, int ne, int nt, int rt) : off(o), num_experts(ne), n_tiles(nt), rows_total(rt) {}
    __device__ bool locate(int tile, int& e_out, int& nt, int& row0, int& rows) {
        while (e < num_experts) {
            const int first = expert_bound(off, e, rows_total);
            const int cnt = max(expert_bound(off, e + 1, rows_total) - first, 0);
            const int parts0 = max(1, (cnt + 255) / 256);
            const int part = ((cnt + parts0 - 1) / parts0 + 31) & ~31;
            const int tiles = cnt > 0 ? ((cnt + part - 1) / part) * n_tiles : 0;
            if (tile < base + tiles) {
                const int local = tile - base, mt = local / n_tiles;
                nt = local - mt * n_tiles;
                row0 = first + mt * part;
                rows = min(part, cnt - mt * part);
                e_out = e;
                return true;
            }
            base += tiles;
            ++e;
        }
        return false;
    }
};

template <bool W_MN, bool SWIGLU>
__global__ void __launch_bounds__(kEmThreads, 1)
grouped_gemm_16_rows_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_a32,
                            const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ CUtensorMap tmap_out, const GroupedMlpParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {  // swizzled TMA tiles need it; the same in both CTAs of a pair
        if (threadIdx.x == 0) record_status(p.status, CAM_ERR_BAD_INDEX, 4, static_cast<int>(smem_u32(smem) & 1023u));
        return;
    }
    constexpr int NS = kErStages;
    uint8_t* stg = smem + NS * kErStageBytes;
    uint8_t* ctrl = stg + kEmStgBytes;
    uint64_t* bar_full = reinterpret_cast<uint64_t*>(ctrl);  // first CTA: bytes of both CTAs' stage have landed
    uint64_t* bar_empty = bar_full + NS;                     // each CTA: the MMAs that read a stage have retired
    uint64_t* bar_tfull = bar_empty + NS;                    // each CTA: the accumulators of a tile are complete
    uint64_t* bar_tempty = bar_tfull + 1;                    // first CTA: both CTAs have drained them
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_tempty + 1);
    volatile uint32_t* abort_flag = tmem_slot + 1;

    const int warp = static_cast<int>(threadIdx.x) >> 5;
    const uint32_t lane = lane_id();
    const uint32_t cta = cluster_cta_rank();  // 0 = first CTA of the pair (issues the MMAs)
    const int pair_id = static_cast<int>(blockIdx.x) >> 1;
    const int num_pairs = static_cast<int>(gridDim.x) >> 1;
    const int nblk = (p.n_dim + 127) / 128;                             // blocks of result columns
    const int n_tiles = SWIGLU ? (nblk + 1) / 2 : (nblk + 3) / 4;
    const int kblocks = (p.k_dim + 63) / 64;

    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&bar_full[s], 1);
            mbar_init(&bar_empty[s], 1);
        }
        mbar_init(bar_tfull, 1);
        mbar_init(bar_tempty, 2 * (kEmEpiThreads / 32));
        *abort_flag = 0u;
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, kEmTmemCols);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();  // both CTAs' barriers are initialised before anything signals them
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    pdl_wait();
    pdl_release();
    PartWalker w(p.expert_offsets, p.num_experts, n_tiles, p.rows);
    int e, nt, row0, rows;
    // result columns of this CTA's two blocks; past the last block nothing is loaded that exists (zeros) and nothing is stored
    auto col_lo = [&]() { return SWIGLU ? (2 * nt + static_cast<int>(cta)) * 128 : (4 * nt + 2 * static_cast<int>(cta)) * 128; };

    if (warp < kEmEpiWarp0) {
        reg_dealloc<kEmCtrlRegs>();
        const uint32_t abort_at = smem_u32(tmem_slot + 1);
        const uint32_t full_at = smem_u32(bar_full), empty_at = smem_u32(bar_empty);
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
            for (int tile = pair_id; !aborted(abort_flag) && w.locate(tile, e, nt, row0, rows); tile += num_pairs) {
                const int half = ((rows + 31) & ~31) / 2;  // rows of the tile in each CTA
                const int pieces = (half + 31) / 32;
                const uint32_t bytes = 2u * (2u * kEmTile + static_cast<uint32_t>(pieces) * 4096u);
                const int my_row = row0 + static_cast<int>(cta) * half, lo = col_lo();
                for (int kb = 0; kb < kblocks; ++kb) {
                    const uint32_t s = ring.s;
                    if (!ready) mbar_wait_warp(empty_at + 8u * s, ring.ph ^ 1u, abort_at);
                    ring.next(NS);
                    ready = mbar_test(empty_at + 8u * ring.s, ring.ph ^ 1u);
                    if (leader) {
                        uint8_t* sw = smem + s * kErStageBytes;
                        uint8_t* sr = sw + 2 * kEmTile;
                        const uint32_t bar = full0 + 8u * s;
                        if (cta == 0) mbar_arrive_expect_tx(&bar_full[s], bytes);
                        if constexpr (W_MN) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) tma_load_3d_pair(sw + i * 8192, &tmap_b, bar, lo * 2 + i * 128, kb * 64, e);
                        } else {
                            tma_load_3d_pair(sw, &tmap_b, bar, kb * 128, lo, e);
                            tma_load_3d_pair(sw + kEmTile, &tmap_b, bar, kb * 128, SWIGLU ? p.n_dim + lo : lo + 128, e);
                        }
                        if (pieces == 4) tma_load_2d_pair(sr, &tmap_a, bar, kb * 128, my_row);
                        else for (int i = 0; i < pieces; ++i) tma_load_2d_pair(sr + i * 4096, &tmap_a32, bar, kb * 128, my_row + i * 32);
                    }
                    __syncwarp();
                }
            }
            if (leader && *abort_flag) record_status(p.status, CAM_ERR_TIMEOUT_PIPELINE, 0, 1);
        } else if (warp == 1 && cta == 0) {
            // ------------------------------------------------------------ MMA issuer (first CTA only)
            const bool leader = elect_one();
            Ring ring;
            uint32_t tcount = 0, ready = 0u;
            for (int tile = pair_id; !aborted(abort_flag) && w.locate(tile, e, nt, row0, rows); tile += num_pairs, ++tcount) {
                const uint32_t n = static_cast<uint32_t>((rows + 31) & ~31);
                const uint32_t idesc = umma_idesc(2 * BM, 0, 1u, p.fp16 ? 0u : 1u) | ((n >> 3) << 17) | (W_MN ? 1u << 15 : 0u);
                // both epilogues must have drained the accumulators
                mbar_wait_warp(smem_u32(bar_tempty), (tcount & 1u) ^ 1u, abort_at);
                tc_fence_after_sync();
                for (int kb = 0; kb < kblocks; ++kb) {
                    const uint32_t s = ring.s;
                    if (!ready) mbar_wait_warp(full_at + 8u * s, ring.ph, abort_at);
                    tc_fence_after_sync();
                    ring.next(NS);
                    ready = mbar_test(full_at + 8u * ring.s, ring.ph);
                    const uint32_t sw = smem_u32(smem) + s * kErStageBytes;
                    const uint64_t lo = W_MN ? umma_desc_mn_sw128(sw) : umma_desc_k_sw128(sw);
                    const uint64_t hi = W_MN ? umma_desc_mn_sw128(sw + kEmTile) : umma_desc_k_sw128(sw + kEmTile);
                    const uint64_t rd = umma_desc_k_sw128(sw + 2 * kEmTile);
                    if (leader) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {  // 16 of the contraction: 32 bytes of a row, or 16 rows of 128 bytes
                            tc_mma_16_pair(tmem_base, lo + (W_MN ? 128u : 2u) * k, rd + 2u * k, idesc, (kb | k) ? 1u : 0u);
                            tc_mma_16_pair(tmem_base + 256u, hi + (W_MN ? 128u : 2u) * k, rd + 2u * k, idesc, (kb | k) ? 1u : 0u);
                        }
                        tc_commit_both(empty_at + 8u * s);
                    }
                    __syncwarp();
                }
                if (leader) tc_commit_both(smem_u32(bar_tfull));
                __syncwarp();
            }
            if (leader && *abort_flag) record_status(p.status, CAM_ERR_TIMEOUT_PIPELINE, 1, static_cast<int>(tcount));
        }
    } else {
        reg_alloc<kEmEpiRegs>();
        // ---------------------------------------------------------------- epilogue warps: a result column per lane
        const int ew = warp - kEmEpiWarp0;
        const int q = warp & 3;   // TMEM lane quarter this warp may read
        const int cq = ew >> 2;   // which 32 rows of each 128
        const int f = q * 32 + static_cast<int>(lane);  // column inside a block of 128
        const bool fp16 = p.fp16 != 0;
        // Two warps share 32 rows x 64 columns, which go through shared memory and leave as one tensor copy; rows of a block of 32 that
        // ends inside it are stored from registers.  w16 holds rows (2 i, 2 i + 1) of this thread's 32, which start at row r0 + 32 cq
        // of the tile; column c of the result is the block's first.
        const int box = cq * 2 + (q >> 1), x = f & 63;
        uint8_t* stage = stg + box * 4096;
        const bool issues = (q & 1) == 0 && lane == 0;
        auto push = [&](const uint32_t* w16, int r0, int c) {
            const int first = r0 + cq * 32;
            if (first >= rows || c + (q >> 1) * 64 >= p.n_dim) return;  // the same in both warps
            if (first + 32 <= rows) {
                if (issues) bulk_wait_group_read<0>();  // the copy that reads this buffer is done with it
                named_bar_sync(1 + box, 64);
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    *reinterpret_cast<uint16_t*>(stage + j * 128 + (((x >> 3) ^ (j & 7)) << 4) + (x & 7) * 2) = static_cast<uint16_t>(w16[j >> 1] >> (16 * (j & 1)));
                fence_proxy_async_smem();
                named_bar_sync(1 + box, 64);
                if (issues) {
                    tma_store_2d(&tmap_out, smem_u32(stage), (c + (q >> 1) * 64) * 2, row0 + first);
                    bulk_commit_group();
                }
            } else if (c + f < p.n_dim) {
                uint16_t* to = reinterpret_cast<uint16_t*>(p.out) + static_cast<size_t>(row0 + first) * p.n_dim + c + f;
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (first + j < rows) to[static_cast<size_t>(j) * p.n_dim] = static_cast<uint16_t>(w16[j >> 1] >> (16 * (j & 1)));
            }
        };
        uint32_t tcount = 0;
        for (int tile = pair_id; w.locate(tile, e, nt, row0, rows); tile += num_pairs, ++tcount) {
            const uint32_t t0 = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(cq * 32);
            const int c_lo = col_lo();
            const bool two = rows > 128;  // a second 128 rows: the same in every thread of the CTA
            const bool has[2] = {cq * 32 < rows, 128 + cq * 32 < rows};  // columns past the tile's rows were not written
            auto hand_back = [&]() {  // what this warp needs of the accumulators is in registers
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if (cta == 0) mbar_arrive(bar_tempty);
                    else mbar_arrive_cluster(map_to_cta(bar_tempty, 0));
                }
            };
            epilogue_wait(bar_tfull, tcount & 1u, abort_flag, 64u);
            tc_fence_after_sync();
            if constexpr (SWIGLU) {
                uint32_t act[2][16];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (has[h]) {
                        uint32_t v0[32], v1[32];
                        tmem_ld_32x32b_x32(t0 + h * 128u, v0);
                        tmem_ld_32x32b_x32(t0 + h * 128u + 256u, v1);
                        tc_wait_ld_regs(v0);
                        tc_wait_ld_regs(v1);
                        if (p.gate_up != nullptr && c_lo + f < p.n_dim) {
                            const size_t pitch = 2 * static_cast<size_t>(p.n_dim);
                            const int left = rows - (h * 128 + cq * 32);
                            float* gu = p.gate_up + static_cast<size_t>(row0 + h * 128 + cq * 32) * pitch + c_lo + f;
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                if (j < left) {
                                    gu[j * pitch] = __uint_as_float(v0[j]);
                                    gu[j * pitch + p.n_dim] = __uint_as_float(v1[j]);
                                }
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            const float g0 = __uint_as_float(v0[j]), g1 = __uint_as_float(v0[j + 1]);
                            act[h][j >> 1] = pack16(g0 * sigmoid_fast(g0) * __uint_as_float(v1[j]), g1 * sigmoid_fast(g1) * __uint_as_float(v1[j + 1]), fp16);
                        }
                    }
                }
                hand_back();
                if (c_lo < p.n_dim) {  // the same in every thread of the CTA
                    push(act[0], 0, c_lo);
                    if (two) push(act[1], 128, c_lo);
                }
            } else {
                uint32_t res[4][16];  // [128 rows][block]
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (has[i >> 1]) {
                        uint32_t v[32];
                        tmem_ld_32x32b_x32(t0 + (i >> 1) * 128u + (i & 1) * 256u, v);
                        tc_wait_ld_regs(v);
#pragma unroll
                        for (int j = 0; j < 32; j += 2) res[i][j >> 1] = pack16(__uint_as_float(v[j]), __uint_as_float(v[j + 1]), fp16);
                    }
                }
                hand_back();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = c_lo + (i & 1) * 128;
                    if (c < p.n_dim && (i < 2 || two)) push(res[i], (i >> 1) * 128, c);
                }
            }
        }
        if ((q & 1) == 0) bulk_wait_group<0>();  // everything this thread sent has been written
        if (*abort_flag) record_status(p.status, CAM_ERR_TIMEOUT_PIPELINE, 2, static_cast<int>(tcount));
        if (!SWIGLU)  // rows of no expert; act and dgu of such rows are read by nothing
            zero_loose_rows(p.out, p.n_dim / 8, p.expert_offsets, p.num_experts, p.rows, static_cast<int>(threadIdx.x) - kEmEpiWarp0 * 32, kEmEpiThreads);
    }

    // ------------------------------------------------------------------ teardown
    abort_drain(abort_flag);
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();  // the other CTA may still read this CTA's shared memory or signal its barriers
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem_base, kEmTmemCols);
    }
}

}  // namespace cam

namespace {

template <bool W_MN, bool SWIGLU>
int launch_rows(const cam::GroupedMlpParams* p, const CUtensorMap* ta, const CUtensorMap* ta32, const CUtensorMap* tb, const CUtensorMap* tout, cudaStream_t stream) {
    static cam::PairLimit limit;
    const int64_t nblk = (p->n_dim + 127) / 128, n_tiles = SWIGLU ? (nblk + 1) / 2 : (nblk + 3) / 4;
    // parts of an expert's rows: at most one beyond the full ones
    const int64_t parts = p->rows / 256 + (p->rows < p->num_experts ? p->rows : p->num_experts);
    return cam::launch_pairs(limit, cam::grouped_gemm_16_rows_kernel<W_MN, SWIGLU>, cam::kEmThreads, cam::kErSmem, parts * n_tiles, stream, *ta, *ta32, *tb, *tout, *p);
}

template <bool DW>
int launch_square(const cam::GroupedMlpParams* p, const CUtensorMap* ta, const CUtensorMap* ta32, const CUtensorMap* tb, const CUtensorMap* tout, cudaStream_t stream) {
    static cam::PairLimit limit;
    const int64_t blocks = DW ? static_cast<int64_t>(p->num_experts) * ((p->m_dim + 255) / 256)
                              : p->rows / 256 + (p->rows < p->num_experts ? p->rows : p->num_experts);
    return cam::launch_pairs(limit, cam::grouped_gemm_16_square_kernel<DW>, cam::kEmThreads, cam::kEmSmem, blocks * ((p->n_dim + 255) / 256), stream, *ta, *ta32, *tb, *tout, *p);
}

}  // namespace

extern "C" int cam_launch_grouped_mlp(const cam::GroupedMlpParams* p, int form, const CUtensorMap* tmap_a, const CUtensorMap* tmap_a32,
                                      const CUtensorMap* tmap_b, const CUtensorMap* tmap_out, cudaStream_t stream) {
    switch (form) {
        case cam::kMlpUp: return launch_rows<false, true>(p, tmap_a, tmap_a32, tmap_b, tmap_out, stream);
        case cam::kMlpDown: return launch_rows<false, false>(p, tmap_a, tmap_a32, tmap_b, tmap_out, stream);
        case cam::kMlpDact: return launch_square<false>(p, tmap_a, tmap_a32, tmap_b, tmap_out, stream);
        case cam::kMlpDx: return launch_rows<true, false>(p, tmap_a, tmap_a32, tmap_b, tmap_out, stream);
        case cam::kMlpDw: return launch_square<true>(p, tmap_a, tmap_a32, tmap_b, tmap_out, stream);
    }
    return static_cast<int>(cudaErrorInvalidValue);
}
