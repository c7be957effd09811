// What the grouped products of the stand-alone expert-MLP operators share: the walker over the tiles of ragged experts, the
// zero fill of rows that belong to no expert, the epilogue's staging of 16-bit rows and the launch on CTA pairs.
#pragma once
#include "expert_ops.h"
#include "gemm_common.cuh"

namespace cam {

// Offsets are data on the device: whatever they hold, first and last row of an expert stay inside [0, rows].
__device__ __forceinline__ int expert_bound(const int* off, int i, int rows) { return min(max(__ldg(off + i), 0), rows); }

// Tiles of 256 rows x n_tiles columns of every expert, expert by expert; the columns of a row block are neighbours.
struct PairTileWalker {
    const int* off;
    int num_experts, n_tiles, rows_total;
    int e = 0, base = 0;
    __device__ PairTileWalker(const int* o, int ne, int nt, int rt) : off(o), num_experts(ne), n_tiles(nt), rows_total(rt) {}
    __device__ bool locate(int tile, int& e_out, int& nt, int& row0, int& rows) {
        while (e < num_experts) {
            const int first = expert_bound(off, e, rows_total);
            const int cnt = max(expert_bound(off, e + 1, rows_total) - first, 0);
            const int tiles = ((cnt + 2 * BM - 1) / (2 * BM)) * n_tiles;
            if (tile < base + tiles) {
                const int local = tile - base, mt = local / n_tiles;
                nt = local - mt * n_tiles;
                row0 = first + mt * 2 * BM;
                rows = min(2 * BM, cnt - mt * 2 * BM);
                e_out = e;
                return true;
            }
            base += tiles;
            ++e;
        }
        return false;
    }
};

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
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(2);
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem_bytes);
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
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
    return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, args...));
}

}  // namespace cam
