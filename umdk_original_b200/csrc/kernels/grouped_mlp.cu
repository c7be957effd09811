// Gated feed-forward block of 16-bit experts, forward and backward, on CTA pairs with fp32 accumulators.  For the rows r of
// expert e (w1 [E, 2I, h] with the gate rows first, w2 [E, h, I]):
//   up      g = x Wg^T, u = x Wu^T, act = silu(g) u            one kernel: both projections, the activation, the product
//   down    y = act W2^T
//   dact    da = dy W2, s = 1 / (1 + e^-g):  dg = da u s (1 + g (1 - s)),  du = da g s    one kernel, da never leaves it
//   dx      dx = dg Wg + du Wu = dgu W1
//   dw      dW2 = dy^T act,  dW1 = dgu^T x, the sums over the rows of the expert
// What is rounded to 16 bits: act and dgu, because they are operands of the next product, and the results.  Gate and up are
// kept in fp32 for the backward pass and da stays in the accumulator, so that no result is more than one rounding of an
// operand and its own away from the formula.
//
// One pipeline for all five: K-blocks of 64 values (128 bytes) come by TMA into a ring of six stages, each CTA of the pair
// holds 128 rows of A and half of the 256-column B tile, one CTA issues tcgen05.mma.cta_group::2, and the accumulator (256
// columns of tensor memory) is one of two, so that the epilogue of a tile overlaps the MMAs of the next.  An operand whose
// contraction index is not its contiguous one (w2 and w1 of dact and dx, both operands of dw) is loaded as [64 of the
// contraction][64 values] boxes and read by the tensor core in its MN-major form; nothing is transposed in memory.
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
constexpr int kEmStgPitch = 272;
constexpr int kEmStgBytes = 128 * kEmStgPitch;
constexpr int kEmSmem = kEmStages * kEmStageBytes + kEmStgBytes + 1024;
static_assert(kEmSmem <= 232448, "exceeds the shared memory of one CTA");
constexpr uint32_t kEmTmemCols = 512;
// setmaxnreg: the shares must not exceed what the CTA was launched with (checked against ptxas by the build)
constexpr uint32_t kEmLaunchRegs = 96, kEmCtrlRegs = 40, kEmEpiRegs = 104;
static_assert(128 * kEmCtrlRegs + kEmEpiThreads * kEmEpiRegs <= kEmLaunchRegs * kEmThreads,
              "setmaxnreg budget exceeds the registers the CTA owns: the kernel would hang");

static __device__ CamStatus g_mlp_status;

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

// MN-major tile with 128-byte swizzle: chunks of 64 values along M (or N), each [64 of the contraction][128 bytes]; chunks are
// 8192 bytes apart (leading byte offset), groups of 8 of the contraction 1024 bytes (stride byte offset).
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t smem_addr) {
    return static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(8192 >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
           (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}

__device__ __forceinline__ float4 ld_nc_f4(const float* p) {
    const uint4 v = ld_nc_v4(p);
    return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
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

// A_MN / B_MN: the operand's contraction index is its row index in memory.  A_MN is the weight-gradient form.
template <bool A_MN, bool B_MN, int EPI>
__global__ void __launch_bounds__(kEmThreads, 1)
grouped_gemm_16_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_a32,
                       const __grid_constant__ CUtensorMap tmap_b, const GroupedMlpParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {  // swizzled TMA tiles need it; the same in both CTAs of a pair
        if (threadIdx.x == 0) gemm_record_status(&g_mlp_status, CAM_ERR_BAD_INDEX, 4, static_cast<int>(smem_u32(smem) & 1023u));
        return;
    }
    constexpr int NS = kEmStages;
    constexpr bool WGRAD = A_MN, SWIGLU = EPI == kMlpSwiglu, DSWIGLU = EPI == kMlpSwigluBackward;
    static_assert(!A_MN || B_MN, "not a form that is used");
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
    const int n_tiles = SWIGLU ? (p.n_dim + 127) / 128 : (p.n_dim + 255) / 256;

    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&bar_full[s], WGRAD ? 2 : 1);
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
    auto locate = [&](int tile) { return WGRAD ? wg.locate(tile, e, mt, nt, row0, rows) : wr.locate(tile, e, nt, row0, rows); };
    auto kblocks_of = [&]() { return ((WGRAD ? rows : p.k_dim) + 63) / 64; };

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
            // row forms: only 32-row pieces of A that hold rows are loaded; what stays in the other rows of the stage reaches
            // accumulator rows that nobody reads
            auto pieces = [](int r) { return r > 96 ? 4 : r > 0 ? (r + 31) / 32 : 0; };
            for (int tile = pair_id; !aborted(abort_flag) && locate(tile); tile += num_pairs) {
                const int kblocks = kblocks_of();
                const int p0 = pieces(min(rows, BM)), p1 = pieces(rows - BM), mine = cta ? p1 : p0;
                const uint32_t bytes = WGRAD ? 2u * kEmStageBytes : 2u * kEmTile + static_cast<uint32_t>(p0 + p1) * 4096u;
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
                        if (WGRAD && kb == kblocks - 1 && (rows & 63) != 0) {
                            bar = tail_own + 8u * s;
                            mbar_arrive_expect_tx(&bar_tail[s], kEmStageBytes);
                        } else if (cta == 0) {
                            mbar_arrive_expect_tx(&bar_full[s], bytes);
                        } else if (WGRAD) {
                            mbar_arrive_cluster(bar);
                        }
                        if constexpr (WGRAD) {
                            const int r = row0 + kb * 64, ca = (mt * 256 + half * 128) * 2, cb = (nt * 256 + half * 128) * 2;
                            tma_load_2d_pair(sa, &tmap_a, bar, ca, r);
                            tma_load_2d_pair(sa + 8192, &tmap_a, bar, ca + 128, r);
                            tma_load_2d_pair(sb, &tmap_b, bar, cb, r);
                            tma_load_2d_pair(sb + 8192, &tmap_b, bar, cb + 128, r);
                        } else {
                            if constexpr (B_MN) {
                                const int cb = (nt * 256 + half * 128) * 2;
                                tma_load_3d_pair(sb, &tmap_b, bar, cb, kb * 64, e);
                                tma_load_3d_pair(sb + 8192, &tmap_b, bar, cb + 128, kb * 64, e);
                            } else {
                                tma_load_3d_pair(sb, &tmap_b, bar, kb * 128, SWIGLU ? half * p.n_dim + nt * 128 : nt * 256 + half * 128, e);
                            }
                            const int arow = row0 + half * BM;
                            if (mine == 4) tma_load_2d_pair(sa, &tmap_a, bar, kb * 128, arow);
                            else for (int i = 0; i < mine; ++i) tma_load_2d_pair(sa + i * 4096, &tmap_a32, bar, kb * 128, arow + i * 32);
                        }
                    }
                    __syncwarp();
                }
            }
            if (leader && *abort_flag) gemm_record_status(&g_mlp_status, CAM_ERR_TIMEOUT_PIPELINE, 0, 0);
        } else if (warp == 1 && cta == 0) {
            // ------------------------------------------------------------ MMA issuer (first CTA only)
            const bool leader = elect_one();
            // fp32 accumulator; a_major / b_major (bits 15, 16) = 1 for MN-major operands
            const uint32_t idesc = umma_idesc(2 * BM, 256, 1u, p.fp16 ? 0u : 1u) | (A_MN ? 1u << 15 : 0u) | (B_MN ? 1u << 16 : 0u);
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
                    const uint64_t adesc = A_MN ? umma_desc_mn_sw128(sa) : umma_desc_k_sw128(sa);
                    const uint64_t bdesc = B_MN ? umma_desc_mn_sw128(sa + kEmTile) : umma_desc_k_sw128(sa + kEmTile);
                    if (leader) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)  // 16 of the contraction: 32 bytes of a row, or 16 rows of 128 bytes
                            tc_mma_16_pair(tmem_base + b * 256u, adesc + (A_MN ? 128u : 2u) * k, bdesc + (B_MN ? 128u : 2u) * k, idesc, (kb | k) ? 1u : 0u);
                        tc_commit_both(empty_at + 8u * s);
                    }
                    __syncwarp();
                }
                if (leader) tc_commit_both(smem_u32(&bar_tfull[b]));
                __syncwarp();
            }
            if (leader && *abort_flag) gemm_record_status(&g_mlp_status, CAM_ERR_TIMEOUT_PIPELINE, 1, static_cast<int>(tcount));
        } else if (WGRAD && warp == 2) {
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
            if (!ok && lane == 0) gemm_record_status(&g_mlp_status, CAM_ERR_TIMEOUT_PIPELINE, 5, static_cast<int>(it));
        }
    } else {
        reg_alloc<kEmEpiRegs>();
        // ---------------------------------------------------------------- epilogue warps
        const int ew = warp - kEmEpiWarp0;
        const int q = warp & 3;   // TMEM lane quarter this warp may read
        const int cq = ew >> 2;   // which 32-column quarter of each 128-column half
        const int r = q * 32 + static_cast<int>(lane);
        const bool fp16 = p.fp16 != 0;
        uint8_t* srow = stg + r * kEmStgPitch;
        uint32_t tcount = 0;
        // 128 columns of packed values (16 words per thread) go through shared memory and leave as one bulk copy per row, to
        // column c0 of `orow` (null: the row is not stored) of a matrix `width` wide
        auto push = [&](const uint32_t* w16, uint8_t* orow, int c0, int width) {
            if (cq == 0) bulk_wait_group_read<0>();  // the copies that read this buffer are done with it
            named_bar_sync(1, kEmEpiThreads);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<uint4*>(srow + cq * 64 + j * 16) = make_uint4(w16[4 * j], w16[4 * j + 1], w16[4 * j + 2], w16[4 * j + 3]);
            fence_proxy_async_smem();
            named_bar_sync(1, kEmEpiThreads);
            if (cq == 0) {
                if (orow != nullptr) bulk_store_s2g(orow + static_cast<size_t>(c0) * 2, srow, static_cast<uint32_t>(min(128, width - c0)) * 2u);
                bulk_commit_group();
            }
        };
        for (int tile = pair_id; ok && locate(tile); tile += num_pairs, ++tcount) {
            const uint32_t b = tcount & 1u;
            const int first = (WGRAD ? mt * 256 : 0) + static_cast<int>(cta) * BM;  // of this CTA's rows of the tile
            const bool valid = first + r < (WGRAD ? p.m_dim : rows);
            const size_t orow_i = WGRAD ? static_cast<size_t>(e) * p.m_dim + first + r : static_cast<size_t>(row0 + first + r);
            const bool empty = WGRAD && rows == 0;
            if constexpr (DSWIGLU) {
                // this tile's gate and up come from memory while its MMAs run: a line per lane of each block of 32 rows x 32 columns
                const int left = rows - (first + q * 32);
                if (left > 0) {
                    const int n = min(32, left);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int c = nt * 256 + h * 128 + cq * 32;
                        const float* gu = p.gate_up + gate_up_at(static_cast<size_t>(row0 + first + q * 32), n, 0, p.n_dim, c);
                        if (static_cast<int>(lane) < n && c + 32 <= p.n_dim) {
                            asm volatile("prefetch.global.L2 [%0];" ::"l"(gu + lane * 32u));
                            asm volatile("prefetch.global.L2 [%0];" ::"l"(gu + static_cast<size_t>(p.n_dim) * n + lane * 32u));
                        }
                    }
                }
            }
            const uint32_t t0 = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + b * 256u + cq * 32;
            auto hand_back = [&]() {  // what this warp needs of the accumulator is in registers
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if (cta == 0) mbar_arrive(&bar_tempty[b]);
                    else mbar_arrive_cluster(map_to_cta(&bar_tempty[b], 0));
                }
            };
            if constexpr (DSWIGLU) {
                // n_dim = I columns of da; dgu [rows, 2I].  16 columns at a time: their gate and up values are asked for before
                // the accumulator is waited for, or while the 16 before them are worked on.
                const int n = max(1, min(32, rows - (first + q * 32)));
                const float* gu0 = p.gate_up + gate_up_at(static_cast<size_t>(row0 + first + q * 32), n, static_cast<int>(lane), p.n_dim, nt * 256 + cq * 32);
                const size_t up = static_cast<size_t>(p.n_dim) * n;
                float4 g4[4], u4[4];
                auto load = [&](int part) {  // part 0..3: half part / 2, columns 16 (part % 2)
                    const int off = (part >> 1) * 128 + (part & 1) * 16;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool in = valid && nt * 256 + cq * 32 + off + 4 * i < p.n_dim;
                        const float* at = gu0 + (off + 4 * i) * n;
                        g4[i] = in ? ld_nc_f4(at) : make_float4(0, 0, 0, 0);
                        u4[i] = in ? ld_nc_f4(at + up) : make_float4(0, 0, 0, 0);
                    }
                };
                load(0);
                if (!mbar_wait_bounded(&bar_tfull[b], (tcount >> 1) & 1u, abort_flag, 2000000000ull, 64u)) { ok = false; break; }
                tc_fence_after_sync();
                uint8_t* orow = valid ? static_cast<uint8_t*>(p.out) + orow_i * (4 * static_cast<size_t>(p.n_dim)) : nullptr;
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
                            const float gg[4] = {g4[i].x, g4[i].y, g4[i].z, g4[i].w}, uu[4] = {u4[i].x, u4[i].y, u4[i].z, u4[i].w};
                            float a[4], d[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float da = __uint_as_float(v[part * 16 + 4 * i + k]);
                                const float s = sigmoid_fast(gg[k]);
                                a[k] = da * uu[k] * (s * (1.f + gg[k] * (1.f - s)));
                                d[k] = da * (gg[k] * s);
                            }
                            v[part * 8 + 2 * i] = pack16(a[0], a[1], fp16);  // words 0..15: dg; their da has been used
                            v[part * 8 + 2 * i + 1] = pack16(a[2], a[3], fp16);
                            du[part * 8 + 2 * i] = pack16(d[0], d[1], fp16);
                            du[part * 8 + 2 * i + 1] = pack16(d[2], d[3], fp16);
                        }
                        if (2 * h + part < 3) load(2 * h + part + 1);
                    }
                    if (c0 < p.n_dim) {  // the same in every thread of the CTA
                        push(v, orow, c0, p.n_dim);
                        push(du, orow != nullptr ? orow + static_cast<size_t>(p.n_dim) * 2 : nullptr, c0, p.n_dim);
                    }
                }
                continue;
            }
            if (!mbar_wait_bounded(&bar_tfull[b], (tcount >> 1) & 1u, abort_flag, 2000000000ull, 64u)) { ok = false; break; }
            tc_fence_after_sync();
            uint32_t v0[32], v1[32];  // columns cq*32.. of the first 128-column half, same of the second
            tmem_ld_32x32b_x32(t0, v0);
            tmem_ld_32x32b_x32(t0 + 128, v1);
            tc_wait_ld_regs(v0);
            tc_wait_ld_regs(v1);
            hand_back();
            uint8_t* out = static_cast<uint8_t*>(p.out);
            if constexpr (SWIGLU) {
                const int c0 = nt * 128 + cq * 32;
                if (p.gate_up != nullptr && valid) {
                    const int n = min(32, rows - (first + q * 32));
                    float* gu = p.gate_up + gate_up_at(static_cast<size_t>(row0 + first + q * 32), n, static_cast<int>(lane), p.n_dim, c0);
                    const size_t up = static_cast<size_t>(p.n_dim) * n;
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        if (c0 + j < p.n_dim) {  // n_dim is a multiple of 8
                            *reinterpret_cast<uint4*>(gu + j * n) = make_uint4(v0[j], v0[j + 1], v0[j + 2], v0[j + 3]);
                            *reinterpret_cast<uint4*>(gu + up + j * n) = make_uint4(v1[j], v1[j + 1], v1[j + 2], v1[j + 3]);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    const float g0 = __uint_as_float(v0[j]), g1 = __uint_as_float(v0[j + 1]);
                    v0[j >> 1] = pack16(g0 * sigmoid_fast(g0) * __uint_as_float(v1[j]),
                                        g1 * sigmoid_fast(g1) * __uint_as_float(v1[j + 1]), fp16);
                }
                push(v0, valid ? out + orow_i * p.n_dim * 2 : nullptr, nt * 128, p.n_dim);
            } else {
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    v0[j >> 1] = empty ? 0u : pack16(__uint_as_float(v0[j]), __uint_as_float(v0[j + 1]), fp16);
                    v1[j >> 1] = empty ? 0u : pack16(__uint_as_float(v1[j]), __uint_as_float(v1[j + 1]), fp16);
                }
                uint8_t* orow = valid ? out + orow_i * p.n_dim * 2 : nullptr;
                const int c0 = nt * 256;
                push(v0, orow, c0, p.n_dim);
                if (c0 + 128 < p.n_dim) push(v1, orow, c0 + 128, p.n_dim);  // the same in every thread of the CTA
            }
        }
        if (cq == 0) bulk_wait_group<0>();  // every row this thread sent has been written
        if (!ok) gemm_record_status(&g_mlp_status, CAM_ERR_TIMEOUT_PIPELINE, 2, static_cast<int>(tcount));
        if (EPI == kMlpPlain && !WGRAD)  // rows of no expert; act and dgu of such rows are read by nothing
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

template <bool A_MN, bool B_MN, int EPI>
int launch_16(const cam::GroupedMlpParams* p, const CUtensorMap* ta, const CUtensorMap* ta32, const CUtensorMap* tb, cudaStream_t stream) {
    static cam::PairLimit limit;
    const int64_t n_tiles = EPI == cam::kMlpSwiglu ? (p->n_dim + 127) / 128 : (p->n_dim + 255) / 256;
    // row blocks: at most one per expert beyond the full ones
    const int64_t blocks = A_MN ? static_cast<int64_t>(p->num_experts) * ((p->m_dim + 255) / 256)
                                : p->rows / 256 + (p->rows < p->num_experts ? p->rows : p->num_experts);
    return cam::launch_pairs(limit, cam::grouped_gemm_16_kernel<A_MN, B_MN, EPI>, cam::kEmThreads, cam::kEmSmem, blocks * n_tiles, stream, *ta, *ta32, *tb, *p);
}

}  // namespace

extern "C" int cam_launch_grouped_mlp(const cam::GroupedMlpParams* p, int form, const CUtensorMap* tmap_a, const CUtensorMap* tmap_a32,
                                      const CUtensorMap* tmap_b, cudaStream_t stream) {
    switch (form) {
        case cam::kMlpUp: return launch_16<false, false, cam::kMlpSwiglu>(p, tmap_a, tmap_a32, tmap_b, stream);
        case cam::kMlpDown: return launch_16<false, false, cam::kMlpPlain>(p, tmap_a, tmap_a32, tmap_b, stream);
        case cam::kMlpDact: return launch_16<false, true, cam::kMlpSwigluBackward>(p, tmap_a, tmap_a32, tmap_b, stream);
        case cam::kMlpDx: return launch_16<false, true, cam::kMlpPlain>(p, tmap_a, tmap_a32, tmap_b, stream);
        case cam::kMlpDw: return launch_16<true, true, cam::kMlpPlain>(p, tmap_a, tmap_a, tmap_b, stream);
    }
    return static_cast<int>(cudaErrorInvalidValue);
}

extern "C" int cam_mlp_status(CamStatus* out) { return static_cast<int>(cudaMemcpyFromSymbol(out, cam::g_mlp_status, sizeof(CamStatus))); }
