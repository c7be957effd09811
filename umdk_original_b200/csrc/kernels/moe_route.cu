// moe_route: experts and weights of every token from its logits, and the gradient of the logits.
//
//   score = softmax(logits) or sigmoid(logits);  rank = score + bias, or the logits themselves without a bias (the same order)
//   groups: the topk_groups groups whose best rank (or whose two best together) is largest stay in; then the k largest ranks
//   weight = score (over the sum of the chosen scores with `renormalize`) * scale
//
// One warp per token.  A lane holds consecutive experts, so the lowest lane with the maximum holds the lowest index: equal ranks go to
// the lowest expert.  Experts whose logit or bias is -inf cannot be chosen, places that stay empty hold -1 with weight 0.
//
// What is chosen is what the formula says, not what its rounding says: ranks in fp32 decide only where neighbours differ by more than
// their error; a row with closer ones (2 % of rows of 256 experts with sigmoid and bias) is ranked again in 64 bits.  Ranking
// every row so would be four times the instructions of the whole kernel.
#include <math_constants.h>

#include "layer_ops.h"
#include "layer_values.cuh"

namespace cam {

namespace {

// fp32 as an unsigned number of the same order; 0 is below all of them
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);  // -0 becomes +0
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u ^ ((u >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }

// Consecutive logits of a lane; what is past the row is -inf
template <int DT, int VPL>
__device__ __forceinline__ void load_logits(const RouteParams& p, int64_t row, int lane, float* x) {
    const int64_t at = row * p.experts + lane * VPL;
    if (VPL * kBytes<DT> >= 16 && p.vec) {
#pragma unroll
        for (int v = 0; v < VPL * kBytes<DT> / 16; ++v) {
            constexpr int N = 16 / kBytes<DT>;
            if (lane * VPL < p.experts) {
                const uint4 r = load16_stream(static_cast<const char*>(p.logits) + at * kBytes<DT> + v * 16);
                const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (DT == kDtFp32) x[v * N + i] = __uint_as_float(w[i]);
                    else if constexpr (DT == kDtBf16) {
                        x[v * N + 2 * i] = __uint_as_float(w[i] << 16);
                        x[v * N + 2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
                    } else {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                        x[v * N + 2 * i] = f.x;
                        x[v * N + 2 * i + 1] = f.y;
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) x[v * N + i] = -CUDART_INF_F;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPL; ++i) x[i] = lane * VPL + i < p.experts ? load1<DT>(p.logits, at + i) : -CUDART_INF_F;
    }
}

__device__ __forceinline__ float sigmoidf(float x) { return 1.f / (1.f + expf(-x)); }

// How far apart two ranks in fp32 have to be for their order to be that of the exact ranks: a score is good to 2^-20 (expf, a sum of
// up to 1024 terms in a tree, a division), its sum with a bias is rounded once more, a group's score is the sum of two.
__device__ __forceinline__ float margin(float v) { return 0x1p-17f * (1.f + fabsf(v)); }

// A row in 64 bits.  `rank`: experts doubles of this warp.  Lane j < k returns the expert of place j, or -1.
template <int DT>
__device__ __noinline__ int choose_in_64_bits(const RouteParams& p, int64_t row, double* rank) {
    const int lane = threadIdx.x & 31, e = p.experts;
    const int64_t at = row * e;
    double top = -CUDART_INF, sum = 0.0;
    if (!p.sigmoid) {
        for (int i = lane; i < e; i += 32) top = fmax(top, static_cast<double>(load1<DT>(p.logits, at + i)));
        for (int o = 16; o >= 1; o >>= 1) top = fmax(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        for (int i = lane; i < e; i += 32) sum += exp(static_cast<double>(load1<DT>(p.logits, at + i)) - top);
        for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    }
    auto score = [&](double x) { return p.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - top) / sum; };
    uint32_t open = 0xFFFFFFFFu;
    const int size = e / p.groups;
    if (p.topk_groups < p.groups) {
        for (int i = lane; i < e; i += 32) {
            const double x = load1<DT>(p.logits, at + i), b = p.bias != nullptr ? static_cast<double>(__ldg(p.bias + i)) : 0.0;
            rank[i] = x > -CUDART_INF && b > -CUDART_INF ? (p.bias == nullptr && p.group_top == 1 ? x : score(x) + b) : -CUDART_INF;
        }
        __syncwarp();
        double first = -CUDART_INF, second = -CUDART_INF;
        if (lane < p.groups) {
            for (int i = 0; i < size; ++i) {
                const double v = rank[lane * size + i];
                second = v > first ? first : v > second ? v : second;
                first = v > first ? v : first;
            }
        }
        const double mine = p.group_top == 2 && second > -CUDART_INF ? first + second : first;
        int before = 0;
        for (int g = 0; g < p.groups; ++g) {
            const double o = __shfl_sync(0xFFFFFFFFu, mine, g);
            before += o > mine || (o == mine && g < lane);
        }
        open = __ballot_sync(0xFFFFFFFFu, lane < p.groups && mine > -CUDART_INF && before < p.topk_groups);
        __syncwarp();
    }
    for (int i = lane; i < e; i += 32) {
        const double x = load1<DT>(p.logits, at + i), b = p.bias != nullptr ? static_cast<double>(__ldg(p.bias + i)) : 0.0;
        const bool in = x > -CUDART_INF && b > -CUDART_INF && (open >> (p.topk_groups < p.groups ? i / size : 0) & 1u);
        rank[i] = in ? (p.bias == nullptr ? x : score(x) + b) : -CUDART_INF;
    }
    __syncwarp();
    int mine = -1;
    for (int j = 0; j < p.k; ++j) {
        double best = -CUDART_INF;
        int who = 0x7FFFFFFF;
        for (int i = lane; i < e; i += 32) {
            if (rank[i] > best) {
                best = rank[i];
                who = i;
            }
        }
        for (int o = 16; o >= 1; o >>= 1) {
            const double v = __shfl_xor_sync(0xFFFFFFFFu, best, o);
            const int w = __shfl_xor_sync(0xFFFFFFFFu, who, o);
            if (v > best || (v == best && w < who)) {
                best = v;
                who = w;
            }
        }
        if (who == 0x7FFFFFFF) break;
        if (lane == j) mine = who;
        if (lane == 0) rank[who] = -CUDART_INF;
        __syncwarp();
    }
    return mine;
}

template <int VPL>
constexpr int kRouteWarps = VPL >= 16 ? 4 : 8;  // rows of a block

template <int DT, int VPL>
__global__ void __launch_bounds__(kRouteWarps<VPL> * 32) moe_route_kernel(const RouteParams p) {
    extern __shared__ double scratch[];  // experts per warp
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, first = lane * VPL;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kRouteWarps<VPL> + warp;
    pdl_wait();
    pdl_release();
    if (row >= p.rows) return;
    double* mine64 = scratch + warp * p.experts;
    float x[VPL];
    load_logits<DT, VPL>(p, row, lane, x);
    bool nan = false;
#pragma unroll
    for (int i = 0; i < VPL; ++i) nan |= x[i] != x[i];
    nan = __any_sync(0xFFFFFFFFu, nan);
    const bool grouped = p.topk_groups < p.groups, by_score = p.bias != nullptr;
    const bool need_scores = by_score || (grouped && p.group_top == 2);
    float top = 0.f, inv_sum = 0.f;
    if (!p.sigmoid && (need_scores || !p.renormalize)) {
        top = x[0];
#pragma unroll
        for (int i = 1; i < VPL; ++i) top = fmaxf(top, x[i]);
        top = warp_max(top);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < VPL; ++i) sum += expf(x[i] - top);
        inv_sum = 1.f / warp_sum(sum);
    }
    // ranks as ordered numbers, 0 for what cannot be chosen
    uint32_t rank[VPL];
    float value[VPL];  // what a group's score is made of
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        float r = x[i];
        value[i] = x[i];
        if (need_scores) {
            value[i] = p.sigmoid ? sigmoidf(x[i]) : expf(x[i] - top) * inv_sum;
            if (by_score) {
                const float b = first + i < p.experts ? __ldg(p.bias + first + i) : -CUDART_INF_F;
                value[i] = r = b > -CUDART_INF_F ? value[i] + b : -CUDART_INF_F;
            }
        }
        const bool in = x[i] > -CUDART_INF_F && r > -CUDART_INF_F;
        rank[i] = in ? ordered(r) : 0u;
        if (!in) value[i] = -CUDART_INF_F;
    }
    bool unclear = false;
    if (grouped) {
        const int size = p.experts / p.groups, lanes = size / VPL;
        float one = -CUDART_INF_F, two = -CUDART_INF_F;
        const bool in_lanes = size % VPL == 0 && (lanes & (lanes - 1)) == 0;  // whole lanes, a power of two of them
        if (in_lanes) {
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                two = fmaxf(two, fminf(one, value[i]));
                one = fmaxf(one, value[i]);
            }
            for (int o = 1; o < lanes; o <<= 1) {
                const float a = __shfl_xor_sync(0xFFFFFFFFu, one, o), b = __shfl_xor_sync(0xFFFFFFFFu, two, o);
                two = fmaxf(fminf(one, a), fmaxf(two, b));
                one = fmaxf(one, a);
            }
            const int from = min(31, lane * lanes);
            one = __shfl_sync(0xFFFFFFFFu, one, from);
            two = __shfl_sync(0xFFFFFFFFu, two, from);
        } else {
            float* all = reinterpret_cast<float*>(mine64);
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                if (first + i < p.experts) all[first + i] = value[i];
            }
            __syncwarp();
            if (lane < p.groups) {
                int i = lane % size;  // lanes start at different banks
                for (int n = 0; n < size; ++n) {
                    const float v = all[lane * size + i];
                    two = fmaxf(two, fminf(one, v));
                    one = fmaxf(one, v);
                    i = i + 1 == size ? 0 : i + 1;
                }
            }
        }
        const float mine = p.group_top == 2 && two > -CUDART_INF_F ? one + two : one;
        int before = 0;
        for (int g = 0; g < p.groups; ++g) {
            const float o = __shfl_sync(0xFFFFFFFFu, mine, g);
            before += o > mine || (o == mine && g < lane);
        }
        const bool some = lane < p.groups && mine > -CUDART_INF_F, in = some && before < p.topk_groups;
        const uint32_t open = __ballot_sync(0xFFFFFFFFu, in);
        if (need_scores) {
            const uint32_t low = __reduce_min_sync(0xFFFFFFFFu, in ? ordered(mine) : 0xFFFFFFFFu);
            const uint32_t next = __reduce_max_sync(0xFFFFFFFFu, some && !in ? ordered(mine) : 0u);
            if (next != 0u) unclear = unordered(low) - unordered(next) <= margin(unordered(low));
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int g = in_lanes ? lane / lanes : (first + i) / size;
            if (first + i < p.experts && !(open >> g & 1u)) rank[i] = 0u;
        }
    }
    uint32_t best = 0u;
    int at = 0, expert = -1;
    auto pick = [&] {
        best = rank[0];
        at = 0;
#pragma unroll
        for (int i = 1; i < VPL; ++i) {
            at = rank[i] > best ? i : at;
            best = max(best, rank[i]);
        }
    };
    pick();
    uint32_t last = 0u;
    int last_expert = -1;
    // one place more than asked for, to see how far the next one is
    const int turns = by_score ? p.k + 1 : p.k;
    for (int j = 0; j < turns && !unclear; ++j) {
        const uint32_t m = __reduce_max_sync(0xFFFFFFFFu, best);
        if (m == 0u) break;
        const int owner = __ffs(__ballot_sync(0xFFFFFFFFu, best == m)) - 1;
        const int e = __shfl_sync(0xFFFFFFFFu, first + at, owner);
        if (by_score) {
            if (j > 0 && unordered(last) - unordered(m) <= margin(unordered(last))) {
                // experts of the same logit and bias are equal, all others are looked at again
                const int64_t row0 = row * p.experts;
                unclear = __ldg(p.bias + e) != __ldg(p.bias + last_expert) || load1<DT>(p.logits, row0 + e) != load1<DT>(p.logits, row0 + last_expert);
            }
            last = m;
            last_expert = e;
        }
        if (j < p.k && lane == j) expert = e;
        if (lane == owner) {
#pragma unroll
            for (int i = 0; i < VPL; ++i) rank[i] = i == at ? 0u : rank[i];
            pick();
        }
    }
    if (unclear) {
        __syncwarp();
        expert = choose_in_64_bits<DT>(p, row, mine64);
    }
    if (lane >= p.k) expert = -1;
    const float l = expert >= 0 ? load1<DT>(p.logits, row * p.experts + expert) : -CUDART_INF_F;
    float w;
    if (p.renormalize) {
        // relative to the largest chosen one, so that scores that fp32 cannot hold keep their ratios
        float m = warp_max(l);
        if (p.sigmoid) m = fminf(m, 0.f);
        w = expert < 0 ? 0.f : p.sigmoid ? expf(fminf(l, 0.f) - m) / (1.f + expf(-fabsf(l))) : expf(l - m);
        const float sum = warp_sum(w);
        w = expert < 0 ? 0.f : w / sum;
    } else {
        w = expert < 0 ? 0.f : p.sigmoid ? sigmoidf(l) : expf(l - top) * inv_sum;
    }
    if (lane < p.k) {
        p.idx[row * p.k + lane] = expert;
        p.weights[row * p.k + lane] = nan ? CUDART_NAN_F : w * p.scale;
    }
}

// One warp per row: the chosen experts' gradients meet in shared memory, the row leaves in order.
//   renormalised: q = weight / scale, dlogit = scale (dw - sum(dw q)) q, times 1 - score with sigmoid
//   otherwise: softmax scale score (dw - sum(dw score)) over all experts, sigmoid scale dw score (1 - score)
template <int DT>
__global__ void __launch_bounds__(256) moe_route_backward_kernel(const RouteParams p) {
    extern __shared__ float rows[];  // experts per warp
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = p.experts;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + warp;
    pdl_wait();
    pdl_release();
    if (row >= p.rows) return;
    float* mine = rows + warp * e;
    const int64_t row0 = row * e;
    int64_t id = lane < p.k ? __ldg(p.idx + row * p.k + lane) : -1;
    if (id >= e) id = -1;
    const float g = id >= 0 ? __ldg(p.dweights + row * p.k + lane) * p.scale : 0.f;
    const float l = id >= 0 ? load1<DT>(p.logits, row0 + id) : -CUDART_INF_F;
    const bool dense = !p.sigmoid && !p.renormalize;
    float d, along = 0.f, top = 0.f, inv_sum = 0.f;
    if (p.renormalize) {
        float m = warp_max(l);
        if (p.sigmoid) m = fminf(m, 0.f);
        float q = id < 0 ? 0.f : p.sigmoid ? expf(fminf(l, 0.f) - m) / (1.f + expf(-fabsf(l))) : expf(l - m);
        const float sum = warp_sum(q);
        q = id < 0 ? 0.f : q / sum;
        d = (g - warp_sum(g * q)) * q;
        if (p.sigmoid && id >= 0) d *= sigmoidf(-l);
    } else if (p.sigmoid) {
        d = id >= 0 ? g * sigmoidf(l) * sigmoidf(-l) : 0.f;
    } else {
        top = -CUDART_INF_F;
        for (int i = lane; i < e; i += 32) {
            mine[i] = load1<DT>(p.logits, row0 + i);
            top = fmaxf(top, mine[i]);
        }
        top = warp_max(top);
        float sum = 0.f;
        for (int i = lane; i < e; i += 32) sum += mine[i] = expf(mine[i] - top);
        inv_sum = 1.f / warp_sum(sum);
        const float q = id >= 0 ? expf(l - top) * inv_sum : 0.f;
        along = warp_sum(g * q);
        d = g * q;
        // a row of nothing but -inf has no scores
        for (int i = lane; i < e; i += 32) mine[i] = top > -CUDART_INF_F ? -along * mine[i] * inv_sum : 0.f;
    }
    if (!dense) {
        for (int i = lane; i < e; i += 32) mine[i] = 0.f;
    }
    __syncwarp();
    if (id >= 0) atomicAdd(mine + id, d);  // no two places hold one expert, unless the caller made them so
    __syncwarp();
    for (int i = lane; i < e; i += 32) store1<DT>(p.dlogits, row0 + i, mine[i]);
}

template <int DT, int VPL>
int launch_route(const RouteParams& p, cudaStream_t stream) {
    constexpr int warps = kRouteWarps<VPL>;
    const dim3 grid(static_cast<unsigned>((p.rows + warps - 1) / warps));
    return launch_pdl(moe_route_kernel<DT, VPL>, grid, warps * 32, static_cast<size_t>(warps) * p.experts * sizeof(double), stream, p);
}

template <int DT>
int launch_route_type(RouteParams p, cudaStream_t stream) {
    int vpl = 1;
    while (vpl * 32 < p.experts) vpl *= 2;
    // pieces of 16 bytes: a lane's share is whole ones and so is the row
    p.vec = p.experts % vpl == 0 && vpl * kBytes<DT> % 16 == 0 && p.experts * kBytes<DT> % 16 == 0 && aligned16(p.logits);
    switch (vpl) {
        case 1: return launch_route<DT, 1>(p, stream);
        case 2: return launch_route<DT, 2>(p, stream);
        case 4: return launch_route<DT, 4>(p, stream);
        case 8: return launch_route<DT, 8>(p, stream);
        case 16: return launch_route<DT, 16>(p, stream);
        default: return launch_route<DT, 32>(p, stream);
    }
}

template <int DT>
int launch_backward_type(const RouteParams& p, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>((p.rows + 7) / 8));
    return launch_pdl(moe_route_backward_kernel<DT>, grid, 256, static_cast<size_t>(8) * p.experts * sizeof(float), stream, p);
}

}  // namespace

}  // namespace cam

extern "C" int cam_launch_moe_route(const cam::RouteParams* p, int dtype, cudaStream_t stream) {
    using namespace cam;
    return dtype == kDtBf16 ? launch_route_type<kDtBf16>(*p, stream) : dtype == kDtFp16 ? launch_route_type<kDtFp16>(*p, stream) : launch_route_type<kDtFp32>(*p, stream);
}

extern "C" int cam_launch_moe_route_backward(const cam::RouteParams* p, int dtype, cudaStream_t stream) {
    using namespace cam;
    return dtype == kDtBf16 ? launch_backward_type<kDtBf16>(*p, stream) : dtype == kDtFp16 ? launch_backward_type<kDtFp16>(*p, stream) : launch_backward_type<kDtFp32>(*p, stream);
}
