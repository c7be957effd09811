// moe_group_rows / moe_ungroup_rows: rows of tokens sorted by expert, the experts' results brought back with their weights, and the
// gradients of both.
//
// Rows of one expert keep the order of their (token, choice) pairs, so the result never depends on timing.  The sort is a counting
// sort by one cluster: every warp counts a stretch of pairs (lanes with the same expert find each other with a ballot per bit of its
// index), sums over warps, blocks and experts give every pair its row.  Everything else is bound by memory: a token is read once and written
// to its k rows, or its k rows are read and summed, whole sectors per thread.  8192 tokens of 4096 bf16 to 8 of 128 experts, 604 MB each way:
// sort and copy 106 us, back 92 us (the copy rate), gradients of rows and weights 179 us (1.14 GB, 0.97 of it).
#include <cooperative_groups.h>

#include "launch.h"
#include "layer_ops.h"
#include "layer_values.cuh"

namespace cg = cooperative_groups;

namespace cam {

namespace {

constexpr int kFewPairs = 2048, kFewCompares = 1 << 19;
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortBlocks = 8;

// Row of every pair (slots, -1 without an expert) and first row of every expert, by one cluster.  Shared memory: counts
// [warps][experts], totals and bases [experts].  A warp holds kHeld pairs per lane in registers from the count to the end; more than that
// (65536 pairs in all) go through memory in between.  With a copy of 16 bytes per row behind it, 32768 pairs take 10 us, 65536 13 us.
constexpr int kHeld = 8;

// Lanes with the same value of `bits` bits.  match.any takes the time of a few hundred instructions where values differ: 65536 pairs in 16.5
// us instead of 12.7.
__device__ __forceinline__ uint32_t same_lanes(uint32_t v, int bits) {
    uint32_t same = 0xFFFFFFFFu;
    for (int b = 0; b < bits; ++b) {
        const uint32_t set = __ballot_sync(0xFFFFFFFFu, v >> b & 1u);
        same &= v >> b & 1u ? set : ~set;
    }
    return same;
}

__global__ void __launch_bounds__(kSortThreads) sort_pairs_kernel(const GroupRowsParams p) {
    extern __shared__ int counts[];
    __shared__ int warp_total[kSortWarps];
    cg::cluster_group cluster = cg::this_cluster();
    const int e = p.experts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = static_cast<int>(cluster.block_rank()), blocks = static_cast<int>(cluster.num_blocks());
    int* total = counts + kSortWarps * e;
    int* base = total + e;
    int* mine = counts + warp * e;
    const int64_t pairs = p.tokens * p.k;
    const int64_t share = (pairs + static_cast<int64_t>(blocks) * kSortThreads - 1) / (static_cast<int64_t>(blocks) * kSortThreads) * 32;
    const int64_t begin = (static_cast<int64_t>(rank) * kSortWarps + warp) * share;
    const int64_t end = begin + share < pairs ? begin + share : pairs;
    const bool held = share <= 32 * kHeld;
    const int bits = 32 - __clz(e);
    for (int i = lane; i < e; i += 32) mine[i] = 0;
    __syncwarp();
    pdl_wait();
    pdl_release();
    int id[kHeld], place[kHeld];
    for (int64_t at = begin; at < end; at += 32 * kHeld) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
            const int64_t i = at + u * 32 + lane;
            id[u] = i < end ? load_expert_id(p.idx, p.idx_i64, static_cast<size_t>(i)) : -1;
            if (id[u] >= e) id[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
            if (at + u * 32 >= end) break;
            const uint32_t same = same_lanes(static_cast<uint32_t>(id[u] < 0 ? e : id[u]), bits);
            place[u] = id[u] >= 0 ? mine[id[u]] + __popc(same & ((1u << lane) - 1u)) : -1;
            __syncwarp();
            if (id[u] >= 0 && (same >> lane) == 1u) mine[id[u]] = place[u] + 1;  // the last of them
            __syncwarp();
            const int64_t i = at + u * 32 + lane;
            if (!held && i < end) p.slots[i] = place[u];
        }
    }
    __syncthreads();
    const int x = threadIdx.x;
    int sum = 0;
    if (x < e) {
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            const int c = counts[w * e + x];
            counts[w * e + x] = sum;
            sum += c;
        }
        total[x] = sum;
    }
    int lower = 0, all = sum;
    if (blocks > 1) {
        cluster.sync();
        if (x < e) {
            all = 0;
#pragma unroll
            for (int b = 0; b < kSortBlocks; ++b) {
                const int c = b < blocks ? cluster.map_shared_rank(total, b)[x] : 0;
                lower += b < rank ? c : 0;
                all += c;
            }
        }
    }
    // exclusive sums over the experts
    int upto = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) warp_total[warp] = upto;
    __syncthreads();
    int before = lane < warp ? warp_total[lane] : 0;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
    const int start = before + upto - all;
    if (x < e) {
        base[x] = start + lower;
        if (rank == 0) {
            p.offsets[x] = start;
            if (x == e - 1) p.offsets[e] = start + all;
        }
    }
    __syncthreads();
    if (held) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
            const int64_t i = begin + u * 32 + lane;
            if (i < end) p.slots[i] = id[u] >= 0 ? place[u] + mine[id[u]] + base[id[u]] : -1;
        }
    } else {
        for (int64_t at = begin; at < end; at += 32 * kHeld) {
#pragma unroll
            for (int u = 0; u < kHeld; ++u) {
                const int64_t i = at + u * 32 + lane;
                id[u] = i < end ? load_expert_id(p.idx, p.idx_i64, static_cast<size_t>(i)) : -1;
                place[u] = i < end ? p.slots[i] : -1;
            }
#pragma unroll
            for (int u = 0; u < kHeld; ++u) {
                const int64_t i = at + u * 32 + lane;
                if (i < end && place[u] >= 0) p.slots[i] = place[u] + mine[id[u]] + base[id[u]];
            }
        }
    }
    if (blocks > 1) cluster.sync();  // nobody leaves while its totals are read
}

// How rows are copied: in pieces of 16 bytes, or (ES: bytes of an element) where they start anywhere, in the pieces of each destination row
constexpr int kPieces16 = 0;

template <int ES>
__device__ __host__ __forceinline__ int64_t pieces_of(int64_t row_bytes) { return ES == kPieces16 ? row_bytes / 16 : (row_bytes + 15 + 15) / 16; }

// Items of a token: the pieces of its row, then its scales
template <int ES>
__device__ __forceinline__ void copy_item(const GroupRowsParams& p, int64_t token, int64_t c, int64_t pieces, const int* slot) {
    if (c < pieces) {
        const char* x = static_cast<const char*>(p.x);
        char* rows = static_cast<char*>(p.rows);
        if constexpr (ES == kPieces16) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(x) + token * pieces + c);
#pragma unroll 8
            for (int j = 0; j < p.k; ++j) {
                const int s = slot[j];
                if (s >= 0) reinterpret_cast<uint4*>(rows)[s * pieces + c] = v;
            }
        } else {
            const char* hi = x + p.tokens * p.row_bytes;
#pragma unroll 4
            for (int j = 0; j < p.k; ++j) {
                const int s = slot[j];
                if (s < 0) continue;
                char* row = rows + s * p.row_bytes;
                const int64_t at = c * 16 - static_cast<int64_t>(reinterpret_cast<uintptr_t>(row) & 15u);  // in the row
                if (at >= p.row_bytes || at <= -16) continue;
                const uint4 v = load_window(x + token * p.row_bytes + at, x, hi);
                if (at >= 0 && at + 16 <= p.row_bytes) *reinterpret_cast<uint4*>(row + at) = v;
                else store_some<ES>(row + at, v, at < 0 ? static_cast<int>(-at) / ES : 0, p.row_bytes - at < 16 ? static_cast<int>(p.row_bytes - at) / ES : 16 / ES);
            }
        }
    } else {
        const float v = __ldg(p.scales + token * p.scale_cols + (c - pieces));
        for (int j = 0; j < p.k; ++j) {
            const int s = slot[j];
            if (s >= 0) p.row_scales[static_cast<int64_t>(s) * p.scale_cols + (c - pieces)] = v;
        }
    }
}

// Zeros to the rows (and scales) of no expert
template <int ES>
__device__ __forceinline__ void clear_tail(const GroupRowsParams& p, int64_t from, int64_t first, int64_t step) {
    const int64_t pairs = p.tokens * p.k, begin = from * p.row_bytes, end = pairs * p.row_bytes;
    char* rows = static_cast<char*>(p.rows);  // 16-byte aligned
    for (int64_t i = begin / 16 + first; i * 16 < end; i += step) {
        if (i * 16 >= begin && i * 16 + 16 <= end) *reinterpret_cast<uint4*>(rows + i * 16) = make_uint4(0u, 0u, 0u, 0u);
        else if constexpr (ES != kPieces16)
            store_some<ES>(rows + i * 16, make_uint4(0u, 0u, 0u, 0u), begin > i * 16 ? static_cast<int>(begin - i * 16) / ES : 0, end - i * 16 < 16 ? static_cast<int>(end - i * 16) / ES : 16 / ES);
    }
    for (int64_t i = from * p.scale_cols + first; i < pairs * p.scale_cols; i += step) p.row_scales[i] = 0.f;
}

// The sorted pairs' rows.  The first blocks write zeros to the rows of no expert.
template <int ES, class Index>
__global__ void __launch_bounds__(256) group_rows_kernel(const GroupRowsParams p, unsigned zero_blocks) {
    const Index pieces = static_cast<Index>(pieces_of<ES>(p.row_bytes)), items = pieces + static_cast<Index>(p.scale_cols);
    pdl_wait();
    pdl_release();
    if (blockIdx.x < zero_blocks) {
        clear_tail<ES>(p, __ldg(p.offsets + p.experts), static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, static_cast<int64_t>(zero_blocks) * 256);
        return;
    }
    const Index i = static_cast<Index>(blockIdx.x - zero_blocks) * 256 + threadIdx.x;
    if (i >= static_cast<Index>(p.tokens) * items) return;
    const Index token = i / items;
    copy_item<ES>(p, static_cast<int64_t>(token), static_cast<int64_t>(i - token * items), static_cast<int64_t>(pieces), p.slots + static_cast<int64_t>(token) * p.k);
}

// Few pairs, one launch: every block finds the places of its own token's pairs by comparing them with all ids, and `parts` blocks share the
// token's row.  The place of a pair is the number of ids below its own, or equal to it and earlier.
template <int ES>
__global__ void __launch_bounds__(256) group_few_rows_kernel(const GroupRowsParams p, unsigned parts) {
    __shared__ int counts[kLayerMaxTopk + 1];
    __shared__ uint16_t ids[kFewPairs];
    const int pairs = static_cast<int>(p.tokens) * p.k, token = blockIdx.x / parts, part = blockIdx.x % parts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x <= kLayerMaxTopk) counts[threadIdx.x] = 0;
    pdl_wait();
    pdl_release();
    {
        int id[kFewPairs / 256];
#pragma unroll
        for (int u = 0; u < kFewPairs / 256; ++u) id[u] = u * 256 + static_cast<int>(threadIdx.x) < pairs ? load_expert_id(p.idx, p.idx_i64, u * 256 + threadIdx.x) : -1;
#pragma unroll
        for (int u = 0; u < kFewPairs / 256; ++u) ids[u * 256 + threadIdx.x] = static_cast<uint16_t>(id[u] >= 0 && id[u] < p.experts ? id[u] : p.experts);
    }
    __syncthreads();
    for (int j0 = 0; j0 < p.k; j0 += 8) {
        const int pair0 = token * p.k + j0;
        int own[8], count[8], valid = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            own[j] = j0 + j < p.k ? ids[pair0 + j] : p.experts;
            count[j] = 0;
        }
#pragma unroll 4
        for (int i = threadIdx.x; i < pairs; i += 256) {
            const int id = ids[i];
            valid += id < p.experts;
            // below, or equal and earlier
#pragma unroll
            for (int j = 0; j < 8; ++j) count[j] += id < own[j] + (i < pair0 + j ? 1 : 0);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int sum = __reduce_add_sync(0xFFFFFFFFu, count[j]);
            if (lane == 0 && j0 + j < p.k) atomicAdd(counts + j0 + j, own[j] < p.experts ? sum : warp == 0 ? -1 : 0);
        }
        valid = __reduce_add_sync(0xFFFFFFFFu, valid);
        if (lane == 0 && j0 == 0) atomicAdd(counts + kLayerMaxTopk, valid);
    }
    // offsets: a warp per expert, shared out to all blocks
    for (int e = blockIdx.x * 8 + warp; e <= p.experts; e += gridDim.x * 8) {
        int below = 0;
#pragma unroll 8
        for (int i = lane; i < pairs; i += 32) below += ids[i] < e;
        below = __reduce_add_sync(0xFFFFFFFFu, below);
        if (lane == 0) p.offsets[e] = below;
    }
    __syncthreads();
    if (part == 0 && static_cast<int>(threadIdx.x) < p.k) p.slots[token * p.k + threadIdx.x] = counts[threadIdx.x];
    const int64_t pieces = pieces_of<ES>(p.row_bytes), items = pieces + p.scale_cols;
    for (int64_t c = part * 256 + threadIdx.x; c < items; c += parts * 256) copy_item<ES>(p, token, c, pieces, counts);
    if (counts[kLayerMaxTopk] < pairs)
        clear_tail<ES>(p, counts[kLayerMaxTopk], static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, static_cast<int64_t>(gridDim.x) * 256);
}

template <int ES>
int launch_copy(const GroupRowsParams& p, cudaStream_t stream) {
    const int64_t items = pieces_of<ES>(p.row_bytes) + p.scale_cols, blocks = (p.tokens * items + 255) / 256;
    const int64_t zero = sm_count_of_current_device();
    if (blocks + zero > 0x7FFFFFFF) return static_cast<int>(cudaErrorInvalidValue);
    const dim3 grid(static_cast<unsigned>(blocks + zero));
    if (blocks * 256 < 0x7FFFFFFF) return launch_pdl(group_rows_kernel<ES, uint32_t>, grid, 256, 0, stream, p, static_cast<unsigned>(zero));
    return launch_pdl(group_rows_kernel<ES, uint64_t>, grid, 256, 0, stream, p, static_cast<unsigned>(zero));
}

template <int ES>
int launch_few(const GroupRowsParams& p, cudaStream_t stream) {
    // as many blocks per token as fill the SMs twice, of 256 items at least
    const int64_t items = pieces_of<ES>(p.row_bytes) + p.scale_cols, most = (items + 255) / 256;
    const int64_t want = (2 * sm_count_of_current_device() + p.tokens - 1) / p.tokens, parts = want < most ? want : most;
    return launch_pdl(group_few_rows_kernel<ES>, dim3(static_cast<unsigned>(p.tokens * parts)), 256, 0, stream, p, static_cast<unsigned>(parts));
}

int launch_sort(const GroupRowsParams& p, cudaStream_t stream) {
    static SmemLimitCache limit;
    const int smem = (kSortWarps + 2) * p.experts * static_cast<int>(sizeof(int));
    const cudaError_t err = limit.ensure(sort_pairs_kernel, smem);
    if (err != cudaSuccess) return static_cast<int>(err);
    // One block up to 8192 pairs, a cluster of eight beyond.  One block / cluster, with rows of 16 bytes: 8192 pairs of 32 experts 10.7 / 10.5 us, of
    // 256 17.5 / 15.4, 16384 of 256 21 / 11, 32768 37 / 11; 4096 wait for the host either way.
    const unsigned blocks = p.tokens * p.k > 8192 ? kSortBlocks : 1;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2] = {pdl_attribute(), {}};
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = blocks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, sort_pairs_kernel, p));
}

// Values of a row in pieces of B bytes: 32 (whole sectors per thread) or 16
template <int DT, int B>
struct Piece {
    static constexpr int N = B / kBytes<DT>;
    static constexpr int kWords = B / 4;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const void* base, int64_t i) {
        const char* p = static_cast<const char*>(base) + i * kBytes<DT>;
        if constexpr (B == 32) load32(w, p);
        else {
            const uint4 v = load16_stream(p);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        }
    }
    __device__ __forceinline__ void store(void* base, int64_t i) const {
        char* p = static_cast<char*>(base) + i * kBytes<DT>;
        if constexpr (B == 32) store32(p, w);
        else *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0u;
    }
    __device__ __forceinline__ Pair get(int i) const {
        if constexpr (DT == kDtFp32) return pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else if constexpr (DT == kDtBf16) return pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
        else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            return pair(f.x, f.y);
        }
    }
    __device__ __forceinline__ void set(int i, Pair v) {
        const float2 f = split(v);
        if constexpr (DT == kDtFp32) {
            w[2 * i] = __float_as_uint(f.x);
            w[2 * i + 1] = __float_as_uint(f.y);
        } else if constexpr (DT == kDtBf16) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(f.x, f.y);
            w[i] = *reinterpret_cast<const uint32_t*>(&b);
        } else {
            const __half2 b = __floats2half2_rn(f.x, f.y);
            w[i] = *reinterpret_cast<const uint32_t*>(&b);
        }
    }
};

// A piece of its token's rows per thread, weighted and summed in the order of the choices, U of them in flight
template <int DT, int B, int U, class Index>
__global__ void __launch_bounds__(128) ungroup_rows_kernel(const UngroupRowsParams p) {
    using P = Piece<DT, B>;
    constexpr int N = P::N, H = N / 2;
    const Index pieces = static_cast<Index>(p.h / N);
    pdl_wait();
    pdl_release();
    const Index i = static_cast<Index>(blockIdx.x) * 128 + threadIdx.x;
    if (i >= static_cast<Index>(p.tokens) * pieces) return;
    const Index token = i / pieces;
    const int64_t c = static_cast<int64_t>(i - token * pieces) * N, pair0 = static_cast<int64_t>(token) * p.k, to = static_cast<int64_t>(token) * p.h + c;
    Pair acc[H];
#pragma unroll
    for (int v = 0; v < H; ++v) acc[v] = 0ull;
    for (int j0 = 0; j0 < p.k; j0 += U) {
        P row[U];
        float w[U];
        int slot[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            slot[u] = j0 + u < p.k ? __ldg(p.slots + pair0 + j0 + u) : -1;
            if (slot[u] >= p.num_rows) slot[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            row[u].clear();
            if (slot[u] >= 0) row[u].load(p.rows, static_cast<int64_t>(slot[u]) * p.h + c);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = slot[u] < 0 ? 0.f : p.weights != nullptr ? __ldg(p.weights + pair0 + j0 + u) : 1.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const Pair w2 = pair(w[u], w[u]);
#pragma unroll
            for (int v = 0; v < H; ++v) acc[v] = fma2(w2, row[u].get(v), acc[v]);
        }
    }
    P out;
    if (p.residual != nullptr) {
        out.load(p.residual, to);
#pragma unroll
        for (int v = 0; v < H; ++v) acc[v] = add2(acc[v], out.get(v));
    }
#pragma unroll
    for (int v = 0; v < H; ++v) out.set(v, acc[v]);
    out.store(p.out, to);
}

// A piece of sixteen bytes of a row that starts anywhere, as fp32 values
template <int DT>
__device__ __forceinline__ void widen_piece(const uint4& v, Pair* f) {
    Piece<DT, 16> q;
    q.w[0] = v.x, q.w[1] = v.y, q.w[2] = v.z, q.w[3] = v.w;
#pragma unroll
    for (int i = 0; i < Piece<DT, 16>::N / 2; ++i) f[i] = q.get(i);
}
template <int DT>
__device__ __forceinline__ uint4 narrow_piece(const Pair* f) {
    Piece<DT, 16> q;
#pragma unroll
    for (int i = 0; i < Piece<DT, 16>::N / 2; ++i) q.set(i, f[i]);
    return make_uint4(q.w[0], q.w[1], q.w[2], q.w[3]);
}

// The same for rows of odd widths: pieces of the result's rows, the others' at whatever address those columns have.  8192 x 4095 bf16 from 8
// rows each: 157 us, with one value per thread 408.
template <int DT, class Index>
__global__ void __launch_bounds__(256) ungroup_odd_rows_kernel(const UngroupRowsParams p) {
    constexpr int N = 16 / kBytes<DT>, U = 4;
    const Index pieces = static_cast<Index>((p.h + 2 * N - 2) / N);
    pdl_wait();
    pdl_release();
    const Index i = static_cast<Index>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= static_cast<Index>(p.tokens) * pieces) return;
    const Index token = i / pieces;
    const int64_t bytes = static_cast<int64_t>(p.h) * kBytes<DT>, pair0 = static_cast<int64_t>(token) * p.k;
    char* out = static_cast<char*>(p.out) + static_cast<int64_t>(token) * bytes;
    const int64_t at = static_cast<int64_t>(i - token * pieces) * 16 - static_cast<int64_t>(reinterpret_cast<uintptr_t>(out) & 15u);  // in the row
    if (at >= bytes || at <= -16) return;
    const char* rows = static_cast<const char*>(p.rows);
    Pair acc[N / 2];
#pragma unroll
    for (int v = 0; v < N / 2; ++v) acc[v] = 0ull;
    for (int j0 = 0; j0 < p.k; j0 += U) {
        uint4 row[U];
        float w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = j0 + u < p.k ? __ldg(p.slots + pair0 + j0 + u) : -1;
            const bool in = s >= 0 && s < p.num_rows;
            w[u] = !in ? 0.f : p.weights != nullptr ? __ldg(p.weights + pair0 + j0 + u) : 1.f;
            row[u] = in ? load_window(rows + s * bytes + at, rows, rows + p.num_rows * bytes) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const Pair w2 = pair(w[u], w[u]);
            Pair f[N / 2];
            widen_piece<DT>(row[u], f);
#pragma unroll
            for (int v = 0; v < N / 2; ++v) acc[v] = fma2(w2, f[v], acc[v]);
        }
    }
    if (p.residual != nullptr) {
        const char* r = static_cast<const char*>(p.residual);
        Pair f[N / 2];
        widen_piece<DT>(load_window(r + static_cast<int64_t>(token) * bytes + at, r, r + p.tokens * bytes), f);
#pragma unroll
        for (int v = 0; v < N / 2; ++v) acc[v] = add2(acc[v], f[v]);
    }
    const uint4 v = narrow_piece<DT>(acc);
    if (at >= 0 && at + 16 <= bytes) *reinterpret_cast<uint4*>(out + at) = v;
    else store_some<kBytes<DT>>(out + at, v, at < 0 ? static_cast<int>(-at) / kBytes<DT> : 0, bytes - at < 16 ? static_cast<int>(bytes - at) / kBytes<DT> : N);
}

// Sums of eight values over the lanes of a warp: lane 4 j has the sum of value j.  Values are halved between the lanes as they are added:
// 9 exchanges instead of 40.
__device__ __forceinline__ float warp_sums8(const float (&v)[8]) {
    const int lane = threadIdx.x & 31;
    float a[4], b[2], c;
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = (lane & 16 ? v[i + 4] : v[i]) + __shfl_xor_sync(0xFFFFFFFFu, lane & 16 ? v[i] : v[i + 4], 16);
#pragma unroll
    for (int i = 0; i < 2; ++i) b[i] = (lane & 8 ? a[i + 2] : a[i]) + __shfl_xor_sync(0xFFFFFFFFu, lane & 8 ? a[i] : a[i + 2], 8);
    c = (lane & 4 ? b[1] : b[0]) + __shfl_xor_sync(0xFFFFFFFFu, lane & 4 ? b[0] : b[1], 4);
    c += __shfl_xor_sync(0xFFFFFFFFu, c, 2);
    return c + __shfl_xor_sync(0xFFFFFFFFu, c, 1);
}

constexpr int kZeroRange = 4096;  // rows that a block looks after at a time: a bit each
// Slots that such a block reads in all its rounds at most; beyond, they are marked in a map first, which is two launches more.  Looking / map,
// bf16: 98304 rows of 256 29 / 30 us, of 2048 182 / 184; 131072 of 256 (two rounds) 74 / 37; 262144 of 256 297 / 70; 1048576 of 16 16000 / 203.
constexpr int64_t kMostLooks = 1 << 17;

// Which rows a slot names, a bit each, for the blocks that write zeros to the others: one look at the slots by all SMs.
__global__ void __launch_bounds__(256) clear_used_kernel(uint32_t* used, int64_t words) {
    pdl_wait();
    pdl_release();
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i < words) used[i] = 0u;
}
__global__ void __launch_bounds__(256) mark_used_kernel(const int* slots, int64_t pairs, int64_t num_rows, uint32_t* used) {
    pdl_wait();
    pdl_release();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * 1024 + threadIdx.x;
    int s[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) s[u] = first + u * 256 < pairs ? __ldg(slots + first + u * 256) : -1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        if (s[u] >= 0 && s[u] < num_rows) atomicOr(used + s[u] / 32, 1u << (s[u] % 32));
    }
}

// Gradients of rows (weight x gradient of the token) and of weights (row . gradient of the token), a token per warp or block.  The first
// `zero_blocks` write zeros to rows that no token uses: they read p.used, or each marks its share of the rows by looking at all slots.
constexpr int kOddRows = 0;  // B: rows that start anywhere, in pieces of sixteen bytes of each row

template <int DT, int B, int U, bool WARP>
__global__ void __launch_bounds__(256) ungroup_rows_backward_kernel(const UngroupRowsParams p, unsigned zero_blocks, int range) {
    using P = Piece<DT, B == kOddRows ? 16 : B>;
    constexpr int N = P::N, H = N / 2;
    const int64_t bytes = static_cast<int64_t>(p.h) * kBytes<DT>;
    __shared__ float red[8][8];
    __shared__ uint32_t used[kZeroRange / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int t = WARP ? lane : threadIdx.x, threads = WARP ? 32 : blockDim.x, pieces = B == kOddRows ? (p.h + 2 * N - 2) / N : p.h / N;
    pdl_wait();
    pdl_release();
    if (blockIdx.x < zero_blocks) {
        P none;
        none.clear();
        const int64_t pairs = p.tokens * p.k;
        for (int64_t from = static_cast<int64_t>(blockIdx.x) * range; from < p.num_rows; from += static_cast<int64_t>(zero_blocks) * range) {
            const int n = static_cast<int>(p.num_rows - from < range ? p.num_rows - from : range);
            if (p.used != nullptr) {
                for (int i = threadIdx.x; i * 32 < n; i += blockDim.x) used[i] = __ldg(p.used + from / 32 + i);
            } else {
                for (int i = threadIdx.x; i * 32 < n; i += blockDim.x) used[i] = 0u;
                __syncthreads();
                auto mark = [&](int slot) {
                    const int64_t s = slot - from;
                    if (s >= 0 && s < n) atomicOr(used + s / 32, 1u << (s % 32));
                };
                const int64_t fours = aligned16(p.slots) ? pairs / 4 : 0;
#pragma unroll 4
                for (int64_t i = threadIdx.x; i < fours; i += blockDim.x) {
                    const int4 s = __ldg(reinterpret_cast<const int4*>(p.slots) + i);
                    mark(s.x), mark(s.y), mark(s.z), mark(s.w);
                }
                for (int64_t i = 4 * fours + threadIdx.x; i < pairs; i += blockDim.x) mark(__ldg(p.slots + i));
            }
            __syncthreads();
            for (int i = warp; i * 32 < n; i += warps) {
                uint32_t left = ~used[i] & (n - i * 32 < 32 ? (1u << (n - i * 32)) - 1u : 0xFFFFFFFFu);
                while (left != 0u) {
                    const int64_t row = from + i * 32 + __ffs(left) - 1;
                    left &= left - 1u;
                    if constexpr (B == kOddRows) {
                        for (int c = lane; c < p.h; c += 32) store1<DT>(p.drows, row * p.h + c, 0.f);
                    } else {
                        for (int c = lane; c < pieces; c += 32) none.store(p.drows, row * p.h + c * N);
                    }
                }
            }
            __syncthreads();
        }
        return;
    }
    const int64_t block = blockIdx.x - zero_blocks, token = WARP ? block * warps + warp : block;
    if (WARP && token >= p.tokens) return;
    const int64_t pair0 = token * p.k, token0 = token * p.h;
    for (int j0 = 0; j0 < p.k; j0 += U) {
        int slot[U];
        float w[U], dot[8] = {};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = j0 + u < p.k ? __ldg(p.slots + pair0 + j0 + u) : -1;
            slot[u] = s < p.num_rows ? s : -1;
            w[u] = slot[u] < 0 ? 0.f : p.weights != nullptr ? __ldg(p.weights + pair0 + j0 + u) : 1.f;
        }
        if constexpr (B == kOddRows) {
            const char* rows = static_cast<const char*>(p.rows);
            const char* dout = static_cast<const char*>(p.dout);
            // the pieces are those of the rows written, or of those read where none are written
            const uintptr_t base = reinterpret_cast<uintptr_t>(p.drows != nullptr ? static_cast<const char*>(p.drows) : rows);
            for (int c = t; c < pieces; c += threads) {
                uint4 row[U];
                int at[U];  // in the row; past it: nothing
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int64_t row0 = slot[u] * bytes;
                    const int64_t place = static_cast<int64_t>(c) * 16 - static_cast<int64_t>((base + row0) & 15u);
                    at[u] = slot[u] >= 0 && place < bytes && place > -16 ? static_cast<int>(place) : static_cast<int>(bytes);
                    if (p.dweights != nullptr && at[u] < bytes) row[u] = load_window(rows + row0 + at[u], rows, rows + p.num_rows * bytes);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (at[u] >= bytes) continue;
                    const int from = at[u] < 0 ? -at[u] / kBytes<DT> : 0, left = (static_cast<int>(bytes) - at[u]) / kBytes<DT>, to = left < N ? left : N;
                    Pair d[H], f[H];
                    uint4 v = load_window(dout + token * bytes + at[u], dout, dout + p.tokens * bytes);
                    if (from > 0 || to < N) v = keep_some<kBytes<DT>>(v, from, to);
                    widen_piece<DT>(v, d);
                    if (p.dweights != nullptr) {
                        if (from > 0 || to < N) row[u] = keep_some<kBytes<DT>>(row[u], from, to);
                        widen_piece<DT>(row[u], f);
                        Pair sum = 0ull;
#pragma unroll
                        for (int i = 0; i < H; ++i) sum = fma2(d[i], f[i], sum);
                        const float2 e = split(sum);
                        dot[u] += e.x + e.y;
                    }
                    if (p.drows != nullptr) {
                        const Pair w2 = pair(w[u], w[u]);
#pragma unroll
                        for (int i = 0; i < H; ++i) d[i] = mul2(w2, d[i]);
                        const uint4 o = narrow_piece<DT>(d);
                        char* to_row = static_cast<char*>(p.drows) + slot[u] * bytes + at[u];
                        if (from == 0 && to == N) *reinterpret_cast<uint4*>(to_row) = o;
                        else store_some<kBytes<DT>>(to_row, o, from, to);
                    }
                }
            }
        }
        for (int c = B == kOddRows ? pieces : t; c < pieces; c += threads) {
            P d, row[U];
            d.load(p.dout, token0 + c * N);
            if (p.dweights != nullptr) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    row[u].clear();
                    if (slot[u] >= 0) row[u].load(p.rows, static_cast<int64_t>(slot[u]) * p.h + c * N);
                }
            }
            if (p.drows != nullptr) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (slot[u] < 0) continue;
                    const Pair w2 = pair(w[u], w[u]);
                    P out;
#pragma unroll
                    for (int v = 0; v < H; ++v) out.set(v, mul2(w2, d.get(v)));
                    out.store(p.drows, static_cast<int64_t>(slot[u]) * p.h + c * N);
                }
            }
            if (p.dweights != nullptr) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    Pair sum = 0ull;
#pragma unroll
                    for (int v = 0; v < H; ++v) sum = fma2(d.get(v), row[u].get(v), sum);
                    const float2 f = split(sum);
                    dot[u] += slot[u] >= 0 ? f.x + f.y : 0.f;  // an infinity times the zeros of no row is not one
                }
            }
        }
        if (p.dweights == nullptr) continue;
        const float sum = warp_sums8(dot);
        if constexpr (WARP) {
            if ((lane & 3) == 0 && lane / 4 < U && j0 + lane / 4 < p.k) p.dweights[pair0 + j0 + lane / 4] = sum;
        } else {
            if ((lane & 3) == 0) red[lane / 4][warp] = sum;
            __syncthreads();
            if (threadIdx.x < U && j0 + static_cast<int>(threadIdx.x) < p.k) {
                float all = 0.f;
                for (int i = 0; i < warps; ++i) all += red[threadIdx.x][i];
                p.dweights[pair0 + j0 + threadIdx.x] = all;
            }
            __syncthreads();
        }
    }
}

// Bytes of the pieces that all operands can be read in: 32, 16, or 0 for rows that start anywhere
int piece_of(const UngroupRowsParams& p, int bytes) {
    const int64_t row = static_cast<int64_t>(p.h) * bytes;
    if (row % 32 == 0 && aligned32(p.rows) && aligned32(p.residual) && aligned32(p.out) && aligned32(p.dout) && aligned32(p.drows)) return 32;
    return row % 16 == 0 && aligned16(p.rows) && aligned16(p.residual) && aligned16(p.out) && aligned16(p.dout) && aligned16(p.drows) ? 16 : 0;
}

template <int DT, int B, int U>
int launch_ungroup(const UngroupRowsParams& p, cudaStream_t stream) {
    const int64_t n = p.tokens * (p.h / Piece<DT, B>::N), blocks = (n + 127) / 128;
    if (blocks > 0x7FFFFFFF) return static_cast<int>(cudaErrorInvalidValue);
    const dim3 grid(static_cast<unsigned>(blocks));
    return blocks * 128 < 0x7FFFFFFF ? launch_pdl(ungroup_rows_kernel<DT, B, U, uint32_t>, grid, 128, 0, stream, p) : launch_pdl(ungroup_rows_kernel<DT, B, U, uint64_t>, grid, 128, 0, stream, p);
}

// As many rows in flight as a token has, up to eight.  Two / four / eight: 16384 x 2 of 4096 bf16 69 / 71 / 84 us, 8192 x 4 56 / 56 / 60, 8192 x 8
// 96 / 96 / 94.
template <int DT, int B>
int launch_ungroup_piece(const UngroupRowsParams& p, cudaStream_t stream) {
    return p.k <= 2 ? launch_ungroup<DT, B, 2>(p, stream) : p.k <= 4 ? launch_ungroup<DT, B, 4>(p, stream) : launch_ungroup<DT, B, 8>(p, stream);
}

template <int DT>
int launch_ungroup_odd(const UngroupRowsParams& p, cudaStream_t stream) {
    constexpr int N = 16 / kBytes<DT>;
    const int64_t n = p.tokens * ((p.h + 2 * N - 2) / N), blocks = (n + 255) / 256;
    if (blocks > 0x7FFFFFFF) return static_cast<int>(cudaErrorInvalidValue);
    const dim3 grid(static_cast<unsigned>(blocks));
    return blocks * 256 < 0x7FFFFFFF ? launch_pdl(ungroup_odd_rows_kernel<DT, uint32_t>, grid, 256, 0, stream, p) : launch_pdl(ungroup_odd_rows_kernel<DT, uint64_t>, grid, 256, 0, stream, p);
}

template <int DT>
int launch_ungroup_type(const UngroupRowsParams& p, cudaStream_t stream) {
    const int piece = piece_of(p, kBytes<DT>);
    return piece == 32 ? launch_ungroup_piece<DT, 32>(p, stream) : piece == 16 ? launch_ungroup_piece<DT, 16>(p, stream) : launch_ungroup_odd<DT>(p, stream);
}

// Who writes zeros to the rows without a token
struct ZeroPlan {
    int64_t blocks, range, words;  // rows per block and round; words of the map (0: the blocks look at the slots themselves)
};

ZeroPlan zero_plan(int64_t num_rows, int64_t row_bytes, int64_t pairs) {
    if (num_rows == 0) return {0, 32, 0};
    const int64_t sms = sm_count_of_current_device();
    auto plan = [&](int64_t most) {
        // 64 rows a block at least
        int64_t blocks = (num_rows + 63) / 64;
        blocks = blocks < most ? blocks : most < 1 ? 1 : most;
        const int64_t range = ((num_rows + blocks - 1) / blocks + 31) / 32 * 32;
        return ZeroPlan{blocks, range < kZeroRange ? range : kZeroRange, 0};
    };
    // Blocks that look for themselves each read all slots in every round: all together a 64th of what the rows move, or 16 MB, a round.  One
    // block for 1554 rows of 1000: 13 us instead of 4; 148 for 65536 of 4096: 185 instead of 176.
    const int64_t share = row_bytes / 128, few = (1 << 22) / (pairs + 1), by_bytes = share > few ? share : few;
    ZeroPlan p = plan(sms < by_bytes ? sms : by_bytes);
    const int64_t rounds = (num_rows + p.blocks * p.range - 1) / (p.blocks * p.range);
    if (rounds * pairs <= kMostLooks) return p;
    p = plan(sms);
    p.words = (num_rows + 31) / 32;
    return p;
}

template <int DT, int B, int U>
int launch_ungroup_backward(UngroupRowsParams p, cudaStream_t stream) {
    // A warp per token, or a block.  16384 x 4 bf16, rows of 512: 27 / 94 us, of 1024 47 / 106, of 2048 93 / 129; 256 x 8 of 1024 7.3 / 7.2, of 2048
    // 9.0 / 7.5, where there are too few tokens to fill the SMs with warps.
    const bool warp = p.h <= 1024;
    const int64_t tokens = warp ? (p.tokens + 7) / 8 : p.tokens, pairs = p.tokens * p.k;
    const ZeroPlan zero = p.drows != nullptr ? zero_plan(p.num_rows, static_cast<int64_t>(p.h) * kBytes<DT>, pairs) : ZeroPlan{0, 32, 0};
    if (tokens + zero.blocks > 0x7FFFFFFF) return static_cast<int>(cudaErrorInvalidValue);
    if (tokens + zero.blocks == 0) return 0;
    if (zero.words == 0) {
        p.used = nullptr;
    } else {
        int rc = launch_pdl(clear_used_kernel, dim3(static_cast<unsigned>((zero.words + 255) / 256)), 256, 0, stream, p.used, zero.words);
        if (rc == 0) rc = launch_pdl(mark_used_kernel, dim3(static_cast<unsigned>((pairs + 1023) / 1024)), 256, 0, stream, p.slots, pairs, p.num_rows, p.used);
        if (rc != 0) return rc;
    }
    const dim3 grid(static_cast<unsigned>(tokens + zero.blocks));
    return launch_pdl(warp ? ungroup_rows_backward_kernel<DT, B, U, true> : ungroup_rows_backward_kernel<DT, B, U, false>, grid, 256, 0, stream, p, static_cast<unsigned>(zero.blocks), static_cast<int>(zero.range));
}

// Two / four / eight rows in flight: 16384 x 2 of 4096 bf16 108 / 129 / 187 us, 8192 x 4 97 / 96 / 121, 8192 x 8 178 / 176 / 182; gradients of rows
// alone 75 / 88 / 127, 58 / 62 / 80, 99 / 103 / 120.
template <int DT, int B>
int launch_ungroup_backward_piece(const UngroupRowsParams& p, cudaStream_t stream) {
    return p.k <= 2 ? launch_ungroup_backward<DT, B, 2>(p, stream) : p.k <= 4 ? launch_ungroup_backward<DT, B, 4>(p, stream) : launch_ungroup_backward<DT, B, 8>(p, stream);
}

template <int DT>
int launch_ungroup_backward_type(const UngroupRowsParams& p, cudaStream_t stream) {
    // odd widths are bound by instructions: eight rows at a time take 124 registers, 8192 x 4095 bf16 of 8 rows each 406 us; four 309 us
    const int piece = piece_of(p, kBytes<DT>);
    return piece == 32 ? launch_ungroup_backward_piece<DT, 32>(p, stream) : piece == 16 ? launch_ungroup_backward_piece<DT, 16>(p, stream) : launch_ungroup_backward<DT, kOddRows, 4>(p, stream);
}

}  // namespace

}  // namespace cam

extern "C" int cam_launch_group_rows(const cam::GroupRowsParams* p, cudaStream_t stream) {
    using namespace cam;
    const bool whole = p->row_bytes % 16 == 0 && aligned16(p->x) && aligned16(p->rows);
    // Comparing the pairs of every token with all others costs instructions, the sort costs a launch.  One launch / sort and copy: 128 tokens
    // x 8 of 7168 bf16 6.4 / 9.2 us, 777 x 2 of 1000 7.7 / 7.0 us; with the host's part 200 x 8 of 4096 8.2 / 10.8, 256 x 8 of 1024 11.2 / 10.8, 1024 x 2 of 4096
    // 10.8 / 10.9, 2048 x 1 18.1 / 10.7.
    const int64_t pairs = p->tokens * p->k;
    if (pairs > 0 && pairs <= kFewPairs && p->tokens * pairs <= kFewCompares) {
        if (whole) return launch_few<kPieces16>(*p, stream);
        return p->elem_bytes == 4 ? launch_few<4>(*p, stream) : p->elem_bytes == 2 ? launch_few<2>(*p, stream) : launch_few<1>(*p, stream);
    }
    const int rc = launch_sort(*p, stream);
    if (rc != 0 || p->tokens == 0) return rc;
    if (whole) return launch_copy<kPieces16>(*p, stream);
    return p->elem_bytes == 4 ? launch_copy<4>(*p, stream) : p->elem_bytes == 2 ? launch_copy<2>(*p, stream) : launch_copy<1>(*p, stream);
}

extern "C" int cam_launch_ungroup_rows(const cam::UngroupRowsParams* p, int dtype, cudaStream_t stream) {
    using namespace cam;
    return dtype == kDtBf16 ? launch_ungroup_type<kDtBf16>(*p, stream) : dtype == kDtFp16 ? launch_ungroup_type<kDtFp16>(*p, stream) : launch_ungroup_type<kDtFp32>(*p, stream);
}

extern "C" int64_t cam_ungroup_rows_backward_map_words(int64_t num_rows, int h, int dtype, int64_t pairs) {
    using namespace cam;
    return zero_plan(num_rows, static_cast<int64_t>(h) * (dtype == kDtFp32 ? 4 : 2), pairs).words;
}

// `used` (the words above, where there are any) with `drows`
extern "C" int cam_launch_ungroup_rows_backward(const cam::UngroupRowsParams* p, int dtype, cudaStream_t stream) {
    using namespace cam;
    return dtype == kDtBf16 ? launch_ungroup_backward_type<kDtBf16>(*p, stream) : dtype == kDtFp16 ? launch_ungroup_backward_type<kDtFp16>(*p, stream) : launch_ungroup_backward_type<kDtFp32>(*p, stream);
}
