// moe_group_rows / moe_ungroup_rows: rows of tokens sorted by expert, the experts' results brought back with their weights, and the
// gradients of both.
//
// Rows of one expert keep the order of their (token, choice) pairs, so the result never depends on timing.  The sort is a counting
// sort by one cluster: every warp counts a stretch of pairs (lanes with the same expert find each other with match.any), sums
// over warps, blocks and experts give every pair its row.  Everything else is bound by memory: a token is read once and written
// to its k rows, or its k rows are read and summed, 16 bytes per thread and row.
#include <cooperative_groups.h>

#include "launch.h"
#include "layer_ops.h"
#include "layer_values.cuh"

namespace cg = cooperative_groups;

namespace cam {

namespace {

constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortBlocks = 8;

// Row of every pair (slots, -1 without an expert) and first row of every expert.  Shared memory: counts [warps][experts], totals and
// bases [experts].
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
    for (int i = threadIdx.x; i < kSortWarps * e; i += kSortThreads) counts[i] = 0;
    pdl_wait();
    pdl_release();
    __syncthreads();
    constexpr int U = 4;  // loads in flight
    for (int64_t at = begin; at < end; at += 32 * U) {
        int id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = at + u * 32 + lane;
            id[u] = i < end ? load_expert_id(p.idx, p.idx_i64, static_cast<size_t>(i)) : -1;
            if (id[u] < 0 || id[u] >= e) id[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = at + u * 32 + lane;
            const uint32_t same = __match_any_sync(0xFFFFFFFFu, id[u]);
            const int before = id[u] >= 0 ? mine[id[u]] : 0;
            __syncwarp();
            if (id[u] >= 0 && lane == __ffs(same) - 1) mine[id[u]] = before + __popc(same);
            __syncwarp();
            if (i < end) p.slots[i] = id[u] >= 0 ? before + __popc(same & ((1u << lane) - 1u)) : -1;
        }
    }
    __syncthreads();
    const int x = threadIdx.x;
    int sum = 0;
    if (x < e) {
#pragma unroll 8
        for (int w = 0; w < kSortWarps; ++w) {
            const int c = counts[w * e + x];
            counts[w * e + x] = sum;
            sum += c;
        }
        total[x] = sum;
    }
    cluster.sync();
    int lower = 0, all = 0;
    if (x < e) {
        for (int b = 0; b < blocks; ++b) {
            const int c = cluster.map_shared_rank(total, b)[x];
            lower += b < rank ? c : 0;
            all += c;
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
    if (warp == 0) {
        int v = warp_total[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
            if (lane >= o) v += u;
        }
        warp_total[lane] = v;
    }
    __syncthreads();
    const int start = upto - all + (warp > 0 ? warp_total[warp - 1] : 0);
    if (x < e) {
        base[x] = start + lower;
        if (rank == 0) {
            p.offsets[x] = start;
            if (x == e - 1) p.offsets[e] = start + all;
        }
    }
    cluster.sync();  // bases are there; nobody reads another block's totals any more
    for (int64_t at = begin; at < end; at += 32) {
        const int64_t i = at + lane;
        if (i >= end) continue;
        const int id = load_expert_id(p.idx, p.idx_i64, static_cast<size_t>(i));
        if (id >= 0 && id < e) p.slots[i] += mine[id] + base[id];
    }
}

// Items of a token: the pieces of its row, then its scales.  The blocks behind them write zeros to the rows of no expert.
template <class Unit, class Index>
__global__ void __launch_bounds__(256) group_rows_kernel(const GroupRowsParams p, unsigned copy_blocks) {
    const Index units = static_cast<Index>(p.row_bytes / sizeof(Unit)), items = units + static_cast<Index>(p.scale_cols);
    const Index n = static_cast<Index>(p.tokens) * items;
    pdl_wait();
    pdl_release();
    Unit* rows = static_cast<Unit*>(p.rows);
    if (blockIdx.x < copy_blocks) {
        const Index i = static_cast<Index>(blockIdx.x) * 256 + threadIdx.x;
        if (i >= n) return;
        const Index token = i / items, c = i - token * items;
        const int* slot = p.slots + static_cast<int64_t>(token) * p.k;
        if (c < units) {
            const Unit v = __ldg(static_cast<const Unit*>(p.x) + static_cast<int64_t>(token) * units + c);
#pragma unroll 8
            for (int j = 0; j < p.k; ++j) {
                const int s = __ldg(slot + j);
                if (s >= 0) rows[static_cast<int64_t>(s) * units + c] = v;
            }
        } else {
            const float v = __ldg(p.scales + static_cast<int64_t>(token) * p.scale_cols + (c - units));
            for (int j = 0; j < p.k; ++j) {
                const int s = __ldg(slot + j);
                if (s >= 0) p.row_scales[static_cast<int64_t>(s) * p.scale_cols + (c - units)] = v;
            }
        }
        return;
    }
    const int64_t pairs = p.tokens * p.k, from = __ldg(p.offsets + p.experts);
    const int64_t step = static_cast<int64_t>(gridDim.x - copy_blocks) * 256;
    const int64_t first = static_cast<int64_t>(blockIdx.x - copy_blocks) * 256 + threadIdx.x;
    for (int64_t i = from * units + first; i < pairs * units; i += step) rows[i] = Unit{};
    for (int64_t i = from * p.scale_cols + first; i < pairs * p.scale_cols; i += step) p.row_scales[i] = 0.f;
}

template <class Unit>
int launch_copy(const GroupRowsParams& p, cudaStream_t stream) {
    const int64_t items = p.row_bytes / static_cast<int64_t>(sizeof(Unit)) + p.scale_cols, blocks = (p.tokens * items + 255) / 256;
    const int64_t zero = sm_count_of_current_device();
    if (blocks + zero > 0x7FFFFFFF) return static_cast<int>(cudaErrorInvalidValue);
    const dim3 grid(static_cast<unsigned>(blocks + zero));
    if (blocks * 256 < 0x7FFFFFFF) return launch_pdl(group_rows_kernel<Unit, uint32_t>, grid, 256, 0, stream, p, static_cast<unsigned>(blocks));
    return launch_pdl(group_rows_kernel<Unit, uint64_t>, grid, 256, 0, stream, p, static_cast<unsigned>(blocks));
}

int launch_sort(const GroupRowsParams& p, cudaStream_t stream) {
    static SmemLimitCache limit;
    const int smem = (kSortWarps + 2) * p.experts * static_cast<int>(sizeof(int));
    const cudaError_t err = limit.ensure(sort_pairs_kernel, smem);
    if (err != cudaSuccess) return static_cast<int>(err);
    // one block up to 8192 pairs, a cluster of eight beyond
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

// A piece of eight values (VEC) or one value per thread: the k rows of its token, weighted and summed in the order of the choices
template <int DT, bool VEC, class Index>
__global__ void __launch_bounds__(256) ungroup_rows_kernel(const UngroupRowsParams p) {
    constexpr int N = VEC ? 8 : 1, U = DT == kDtFp32 ? 4 : 8;
    const Index pieces = static_cast<Index>(p.h / N), n = static_cast<Index>(p.tokens) * pieces;
    pdl_wait();
    pdl_release();
    const Index i = static_cast<Index>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= n) return;
    const Index token = i / pieces;
    const int64_t c = static_cast<int64_t>(i - token * pieces) * N, pair0 = static_cast<int64_t>(token) * p.k;
    float acc[N];
#pragma unroll
    for (int v = 0; v < N; ++v) acc[v] = 0.f;
    for (int j0 = 0; j0 < p.k; j0 += U) {
        Raw8<DT> raw[VEC ? U : 1];
        float one[U], w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = j0 + u < p.k ? __ldg(p.slots + pair0 + j0 + u) : -1;
            const bool in = s >= 0 && s < p.num_rows;
            w[u] = !in ? 0.f : p.weights != nullptr ? __ldg(p.weights + pair0 + j0 + u) : 1.f;
            if constexpr (VEC) {
                if (in) raw[u] = load8<DT>(p.rows, static_cast<int64_t>(s) * p.h + c);
                else raw[u] = Raw8<DT>{};
            } else {
                one[u] = in ? load1<DT>(p.rows, static_cast<int64_t>(s) * p.h + c) : 0.f;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if constexpr (VEC) {
                float f[8];
                widen8<DT>(raw[u], f);
#pragma unroll
                for (int v = 0; v < 8; ++v) acc[v] = fmaf(w[u], f[v], acc[v]);
            } else {
                acc[0] = fmaf(w[u], one[u], acc[0]);
            }
        }
    }
    const int64_t to = static_cast<int64_t>(token) * p.h + c;
    if constexpr (VEC) {
        if (p.residual != nullptr) {
            float f[8];
            widen8<DT>(load8<DT>(p.residual, to), f);
#pragma unroll
            for (int v = 0; v < 8; ++v) acc[v] += f[v];
        }
        store8<DT>(p.out, to, narrow8<DT>(acc));
    } else {
        if (p.residual != nullptr) acc[0] += load1<DT>(p.residual, to);
        store1<DT>(p.out, to, acc[0]);
    }
}

__global__ void __launch_bounds__(256) mark_rows_kernel(const int* __restrict__ slots, int64_t pairs, uint8_t* used, int64_t num_rows) {
    pdl_wait();
    pdl_release();
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= pairs) return;
    const int s = __ldg(slots + i);
    if (s >= 0 && s < num_rows) used[s] = 1;
}

// Gradients of rows (weight x gradient of the token) and of weights (row . gradient of the token), a token per warp or block.  The
// blocks behind the tokens' write zeros to rows that no token uses.
template <int DT, bool VEC, bool WARP>
__global__ void __launch_bounds__(256) ungroup_rows_backward_kernel(const UngroupRowsParams p, unsigned token_blocks) {
    constexpr int N = VEC ? 8 : 1, U = 8;
    __shared__ float red[U][8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int t = WARP ? lane : threadIdx.x, threads = WARP ? 32 : blockDim.x, pieces = p.h / N;
    pdl_wait();
    pdl_release();
    if (blockIdx.x >= token_blocks) {
        const int64_t step = static_cast<int64_t>(gridDim.x - token_blocks) * warps;
        for (int64_t r = static_cast<int64_t>(blockIdx.x - token_blocks) * warps + warp; r < p.num_rows; r += step) {
            if (p.used[r] != 0) continue;
            for (int c = lane; c < pieces; c += 32) {
                if constexpr (VEC) store8<DT>(p.drows, r * p.h + c * 8, Raw8<DT>{});
                else store1<DT>(p.drows, r * p.h + c, 0.f);
            }
        }
        return;
    }
    const int64_t token = WARP ? static_cast<int64_t>(blockIdx.x) * warps + warp : blockIdx.x;
    if (WARP && token >= p.tokens) return;
    const int64_t pair0 = token * p.k, token0 = token * p.h;
    for (int j0 = 0; j0 < p.k; j0 += U) {
        int64_t row0[U];
        float w[U], dot[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = j0 + u < p.k ? __ldg(p.slots + pair0 + j0 + u) : -1;
            const bool in = s >= 0 && s < p.num_rows;
            row0[u] = in ? static_cast<int64_t>(s) * p.h : -1;
            w[u] = !in ? 0.f : p.weights != nullptr ? __ldg(p.weights + pair0 + j0 + u) : 1.f;
            dot[u] = 0.f;
        }
        for (int c = t; c < pieces; c += threads) {
            float d[N];
            if constexpr (VEC) widen8<DT>(load8<DT>(p.dout, token0 + c * 8), d);
            else d[0] = load1<DT>(p.dout, token0 + c);
            if (p.dweights != nullptr) {
                Raw8<DT> raw[VEC ? U : 1];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if constexpr (VEC) {
                        if (row0[u] >= 0) raw[u] = load8<DT>(p.rows, row0[u] + c * 8);
                        else raw[u] = Raw8<DT>{};
                    } else {
                        dot[u] = fmaf(d[0], row0[u] >= 0 ? load1<DT>(p.rows, row0[u] + c) : 0.f, dot[u]);
                    }
                }
                if constexpr (VEC) {
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        float f[8];
                        widen8<DT>(raw[u], f);
#pragma unroll
                        for (int v = 0; v < 8; ++v) dot[u] = fmaf(d[v], f[v], dot[u]);
                    }
                }
            }
            if (p.drows != nullptr) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (row0[u] < 0) continue;
                    if constexpr (VEC) {
                        float f[8];
#pragma unroll
                        for (int v = 0; v < 8; ++v) f[v] = w[u] * d[v];
                        store8<DT>(p.drows, row0[u] + c * 8, narrow8<DT>(f));
                    } else {
                        store1<DT>(p.drows, row0[u] + c, w[u] * d[0]);
                    }
                }
            }
        }
        if (p.dweights == nullptr) continue;
#pragma unroll
        for (int u = 0; u < U; ++u) dot[u] = warp_sum(dot[u]);
        if constexpr (WARP) {
            if (lane == 0) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (j0 + u < p.k) p.dweights[pair0 + j0 + u] = dot[u];
                }
            }
        } else {
            if (lane == 0) {
#pragma unroll
                for (int u = 0; u < U; ++u) red[u][warp] = dot[u];
            }
            __syncthreads();
            if (threadIdx.x < U && j0 + static_cast<int>(threadIdx.x) < p.k) {
                float sum = 0.f;
                for (int i = 0; i < warps; ++i) sum += red[threadIdx.x][i];
                p.dweights[pair0 + j0 + threadIdx.x] = sum;
            }
            __syncthreads();
        }
    }
}

bool vectors(const UngroupRowsParams& p) {
    return p.h % 8 == 0 && aligned16(p.rows) && aligned16(p.residual) && aligned16(p.out) && aligned16(p.dout) && aligned16(p.drows);
}

template <int DT>
int launch_ungroup_type(const UngroupRowsParams& p, cudaStream_t stream) {
    const bool vec = vectors(p);
    const int64_t n = p.tokens * (vec ? p.h / 8 : p.h), blocks = (n + 255) / 256;
    if (blocks > 0x7FFFFFFF) return static_cast<int>(cudaErrorInvalidValue);
    const dim3 grid(static_cast<unsigned>(blocks));
    if (blocks * 256 < 0x7FFFFFFF)
        return vec ? launch_pdl(ungroup_rows_kernel<DT, true, uint32_t>, grid, 256, 0, stream, p) : launch_pdl(ungroup_rows_kernel<DT, false, uint32_t>, grid, 256, 0, stream, p);
    return vec ? launch_pdl(ungroup_rows_kernel<DT, true, uint64_t>, grid, 256, 0, stream, p) : launch_pdl(ungroup_rows_kernel<DT, false, uint64_t>, grid, 256, 0, stream, p);
}

template <int DT>
int launch_ungroup_backward_type(const UngroupRowsParams& p, cudaStream_t stream) {
    const bool vec = vectors(p);
    const int64_t pairs = p.tokens * p.k;
    if (p.drows != nullptr && pairs > 0) {
        const int rc = launch_pdl(mark_rows_kernel, dim3(static_cast<unsigned>((pairs + 255) / 256)), 256, 0, stream, p.slots, pairs, p.used, p.num_rows);
        if (rc != 0) return rc;
    }
    const bool warp = p.h <= 1024;
    const int64_t tokens = warp ? (p.tokens + 7) / 8 : p.tokens, zero = p.drows != nullptr ? sm_count_of_current_device() : 0;
    if (tokens + zero > 0x7FFFFFFF) return static_cast<int>(cudaErrorInvalidValue);
    const dim3 grid(static_cast<unsigned>(tokens + zero));
    const unsigned nb = static_cast<unsigned>(tokens);
    if (warp) return vec ? launch_pdl(ungroup_rows_backward_kernel<DT, true, true>, grid, 256, 0, stream, p, nb) : launch_pdl(ungroup_rows_backward_kernel<DT, false, true>, grid, 256, 0, stream, p, nb);
    return vec ? launch_pdl(ungroup_rows_backward_kernel<DT, true, false>, grid, 256, 0, stream, p, nb) : launch_pdl(ungroup_rows_backward_kernel<DT, false, false>, grid, 256, 0, stream, p, nb);
}

}  // namespace

}  // namespace cam

extern "C" int cam_launch_group_rows(const cam::GroupRowsParams* p, cudaStream_t stream) {
    using namespace cam;
    const int rc = launch_sort(*p, stream);
    if (rc != 0 || p->tokens == 0) return rc;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(p->x) | reinterpret_cast<uintptr_t>(p->rows) | static_cast<uintptr_t>(p->row_bytes);
    if (bits % 16 == 0) return launch_copy<uint4>(*p, stream);
    if (bits % 4 == 0) return launch_copy<uint32_t>(*p, stream);
    if (bits % 2 == 0) return launch_copy<uint16_t>(*p, stream);
    return launch_copy<uint8_t>(*p, stream);
}

extern "C" int cam_launch_ungroup_rows(const cam::UngroupRowsParams* p, int dtype, cudaStream_t stream) {
    using namespace cam;
    return dtype == kDtBf16 ? launch_ungroup_type<kDtBf16>(*p, stream) : dtype == kDtFp16 ? launch_ungroup_type<kDtFp16>(*p, stream) : launch_ungroup_type<kDtFp32>(*p, stream);
}

extern "C" int cam_launch_ungroup_rows_backward(const cam::UngroupRowsParams* p, int dtype, cudaStream_t stream) {
    using namespace cam;
    return dtype == kDtBf16 ? launch_ungroup_backward_type<kDtBf16>(*p, stream) : dtype == kDtFp16 ? launch_ungroup_backward_type<kDtFp16>(*p, stream) : launch_ungroup_backward_type<kDtFp32>(*p, stream);
}
