// moe_route: experts and weights of every token from its logits, and the gradient of the logits.
//
//   score = softmax(logits) or sigmoid(logits);  rank = score + bias, or the logits themselves without a bias (the same order)
//   groups: the topk_groups groups whose best rank (or whose two best together) is largest stay in; then the k largest ranks
//   weight = score (over the sum of the chosen scores with `renormalize`) * scale
//
// 8, 16 or 32 lanes share a token, each holds up to 32 consecutive experts as sorted 32-bit keys: the upper bits of the rank, and the
// index, so that keys differ and equal ranks go to the lowest expert.  The largest key of the lanes' heads is taken k times.
// Experts whose logit or bias is -inf cannot be chosen, places that stay empty hold -1 with weight 0.
//
// What is chosen is what the formula says, not what its rounding says.  16-bit logits fit the keys as they are.  Otherwise the keys
// only find candidates: k + 1 of them, whose own ranks are then taken exactly (in 64 bits where scores are ranked) and put in order;
// where the next key is so close that it might belong to them, the row is ranked again by the whole warp.
//
// 620 instructions for four tokens of 128 bf16 logits and k = 8 (32768 tokens 9.2 us, 11.5 MB), 1460 for two tokens of 256 fp32 logits with
// sigmoid, bias and 4 of 8 groups (16384 tokens 18 us); a whole warp per token took three times as many.  Bound by latency rather
// than by their issue (1.9 and 2.1 a cycle of 4, five warps a scheduler): of the 10.8 and 9.3 cycles from one to the next a warp waits 3.0 and 1.7
// for logits, 2.0 and 1.7 for shuffles and shared memory, whose rounds depend on one another, and 1.6 and 2.1 for results of arithmetic.  Rows
// of nothing but equal logits cost four times as much (16384 x 256: 12 and 38 us; with bias and groups 18 and 108).
#include <math_constants.h>

#include "layer_ops.h"
#include "layer_values.cuh"

namespace cam {

namespace {

// fp32 as an unsigned number of the same order; 0 is below all of them
__device__ __forceinline__ uint32_t ordered(float v) {
    const int b = __float_as_int(v + 0.f);  // -0 becomes +0
    return static_cast<uint32_t>(b ^ (b >> 31 | INT32_MIN));
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u ^ ((u >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }

// Consecutive logits of a lane; what is past the row is -inf.  SPREAD: where they go one by one, every 32nd instead, so that the lanes'
// accesses lie side by side: gradients of 17885 x 300 fp16 8 us instead of 34.
template <int DT, int VPL, bool SPREAD = false>
__device__ __forceinline__ void load_logits(const RouteParams& p, int64_t row, int lane, float* x) {
    constexpr int kShare = VPL * kBytes<DT>, kWords = kShare / 4;  // of a lane
    const int64_t at = row * p.experts + lane * VPL;
    if (kShare >= 16 && p.vec) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) x[i] = -CUDART_INF_F;
        if (lane * VPL < p.experts) {
            const char* from = static_cast<const char*>(p.logits) + at * kBytes<DT>;
            uint32_t w[kWords > 0 ? kWords : 1];
            if constexpr (kShare >= 32) {
                // whole sectors: two pieces of 16 bytes would fetch them twice
#pragma unroll
                for (int i = 0; i < kWords; i += 8) load32(w + i, from + i * 4);
            } else if constexpr (kShare == 16) {
                const uint4 v = load16_stream(from);
                w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
            }
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                if constexpr (DT == kDtFp32) x[i] = __uint_as_float(w[i]);
                else if constexpr (DT == kDtBf16) {
                    x[2 * i] = __uint_as_float(w[i] << 16);
                    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
                } else {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                    x[2 * i] = f.x;
                    x[2 * i + 1] = f.y;
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int e = SPREAD ? i * 32 + lane : lane * VPL + i;
            x[i] = e < p.experts ? load1<DT>(p.logits, row * p.experts + e) : -CUDART_INF_F;
        }
    }
}

__device__ __forceinline__ float sigmoidf(float x) { return 1.f / (1.f + expf(-x)); }

// Scores that only find candidates and compare groups, from the approximate exponential and reciprocal: relative error of exp(-x)
// (2 + 1.2 |x|) 2^-23, of the reciprocal 2^-23, so a sigmoid is good to 2^-21 (its error shrinks with exp(-|x|) as it grows with |x|).
// A softmax adds the sum's up to 40 roundings: 2^-18.
__device__ __forceinline__ float quick_exp(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}
__device__ __forceinline__ float quick_sigmoid(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.f + quick_exp(-x)));
    return y;
}
// How far apart two ranks have to be for their order to be that of the exact ones: both errors and the rounding of the bias' addition
__device__ __forceinline__ float margin(const RouteParams& p, float v) { return (p.sigmoid ? 0x1p-20f : 0x1p-17f) + 0x1p-22f * fabsf(v); }

__device__ __forceinline__ unsigned long long ordered(double v) {
    const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(v + 0.0));
    return b ^ (b >> 63 ? ~0ull : 1ull << 63);
}

// One copy for all who call it: what is rarely called finds it in the instruction cache.
__device__ __noinline__ double exact_sigmoid(float x) { return 1.0 / (1.0 + exp(-static_cast<double>(x))); }

// A row in 64 bits, by the whole warp.  `rank`: experts doubles.  Lane j < k returns the expert of place j, or -1.
template <int DT>
__device__ __noinline__ int choose_in_64_bits(const RouteParams& p, int64_t row, double* rank) {
    const int lane = threadIdx.x & 31, e = p.experts;
    const int64_t at = row * e;
    double top = -CUDART_INF, sum = 0.0;
    if (!p.sigmoid) {
        for (int i = lane; i < e; i += 32) top = fmax(top, static_cast<double>(load1<DT>(p.logits, at + i)));
        for (int o = 16; o >= 1; o >>= 1) top = fmax(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
#pragma unroll 4
        for (int i = lane; i < e; i += 32) sum += exp(static_cast<double>(load1<DT>(p.logits, at + i)) - top);
        for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    }
    const bool grouped = p.topk_groups < p.groups, scores = p.bias != nullptr || (grouped && p.group_top == 2);
#pragma unroll 4
    for (int i = lane; i < e; i += 32) {
        const double x = load1<DT>(p.logits, at + i), b = p.bias != nullptr ? static_cast<double>(__ldg(p.bias + i)) : 0.0;
        const double score = !scores ? x : p.sigmoid ? exact_sigmoid(static_cast<float>(x)) : exp(x - top) / sum;
        rank[i] = x > -CUDART_INF && b > -CUDART_INF && score + b > -CUDART_INF ? score + b : -CUDART_INF;
    }
    __syncwarp();
    const int size = e / p.groups;
    if (grouped) {
        double first = -CUDART_INF, second = -CUDART_INF;
        if (lane < p.groups) {
#pragma unroll 4
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
        const uint32_t open = __ballot_sync(0xFFFFFFFFu, lane < p.groups && mine > -CUDART_INF && before < p.topk_groups);
        for (int i = lane; i < e; i += 32) {
            if (!(open >> (i / size) & 1u)) rank[i] = -CUDART_INF;
        }
    }
    if (p.bias == nullptr && scores) {  // the groups were by score, the experts are by logit
        for (int i = lane; i < e; i += 32) {
            if (rank[i] > -CUDART_INF) rank[i] = load1<DT>(p.logits, at + i);
        }
    }
    int mine = -1, who = -1;
    unsigned long long best = 0ull;  // of this lane's experts
    auto look = [&] {
        best = 0ull;
#pragma unroll 4
        for (int i = lane; i < e; i += 32) {
            const unsigned long long r = rank[i] > -CUDART_INF ? ordered(rank[i]) : 0ull;
            who = r > best ? i : who;
            best = r > best ? r : best;
        }
    };
    look();
    for (int j = 0; j < p.k; ++j) {
        const uint32_t hi = __reduce_max_sync(0xFFFFFFFFu, static_cast<uint32_t>(best >> 32));
        const bool in = best != 0ull && static_cast<uint32_t>(best >> 32) == hi;
        const uint32_t lo = __reduce_max_sync(0xFFFFFFFFu, in ? static_cast<uint32_t>(best) : 0u);
        const int next = static_cast<int>(__reduce_min_sync(0xFFFFFFFFu, in && static_cast<uint32_t>(best) == lo ? static_cast<uint32_t>(who) : 0x7FFFFFFFu));
        if (next == 0x7FFFFFFF) break;
        if (lane == j) mine = next;
        if (next % 32 == lane) {
            rank[next] = -CUDART_INF;
            look();
        }
        __syncwarp();
    }
    return mine;
}

// The k largest logits of a row one after the other, for rows with many equal ones.  Lane j < k returns the expert of place j, or -1.
template <int DT>
__device__ __noinline__ int choose_by_logit(const RouteParams& p, int64_t row, uint32_t open, float* all) {
    const int lane = threadIdx.x & 31, size = p.experts / p.groups;
    for (int i = lane; i < p.experts; i += 32) {
        const float x = load1<DT>(p.logits, row * p.experts + i);
        all[i] = open >> (p.topk_groups < p.groups ? i / size : 0) & 1u ? x : -CUDART_INF_F;
    }
    __syncwarp();
    int mine = -1;
    for (int j = 0; j < p.k; ++j) {
        uint32_t best = 0u;
        int at = 0;
        for (int i = lane; i < p.experts; i += 32) {
            const uint32_t r = all[i] > -CUDART_INF_F ? ordered(all[i]) : 0u;
            at = r > best ? i : at;
            best = max(best, r);
        }
        const uint32_t m = __reduce_max_sync(0xFFFFFFFFu, best);
        if (m == 0u) break;
        const int e = static_cast<int>(__reduce_min_sync(0xFFFFFFFFu, best == m ? static_cast<uint32_t>(at) : 0xFFFFFFFFu));
        if (lane == j) mine = e;
        if (lane == 0) all[e] = -CUDART_INF_F;
        __syncwarp();
    }
    return mine;
}

template <int L>
__device__ __forceinline__ float seg_max(float v) {
#pragma unroll
    for (int o = L / 2; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}
template <int L>
__device__ __forceinline__ float seg_sum(float v) {
#pragma unroll
    for (int o = L / 2; o >= 1; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// Largest first: odd-even merge sort
template <int N>
__device__ __forceinline__ void sort_down(uint32_t (&v)[N]) {
#pragma unroll
    for (int p = 1; p < N; p *= 2) {
#pragma unroll
        for (int k = p; k >= 1; k /= 2) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int j = i + k;
                if (j < N && (i - k % p) >= 0 && (i - k % p) / k % 2 == 0 && i / (2 * p) == j / (2 * p)) {
                    const uint32_t hi = max(v[i], v[j]), lo = min(v[i], v[j]);
                    v[i] = hi;
                    v[j] = lo;
                }
            }
        }
    }
}

// Which of the L lanes' groups stay open, a bit each, by the scores that the lanes hold
template <int L, class T>
__device__ __forceinline__ uint32_t best_groups(const RouteParams& p, T mine, bool some) {
    const int sub = threadIdx.x % L;
    int before = 0;
    for (int g = 0; g < p.groups; ++g) {
        const T o = __shfl_sync(0xFFFFFFFFu, mine, g, L);
        before += o > mine || (o == mine && g < sub);
    }
    return __ballot_sync(0xFFFFFFFFu, some && before < p.topk_groups) >> (threadIdx.x & 31 & ~(L - 1)) & (L == 32 ? 0xFFFFFFFFu : (1u << (L & 31)) - 1u);
}

// The groups that stay open, a bit each, from what their experts are worth; the L lanes of a token call it together.  `unclear`: the border
// between the groups is closer than the scores are good for.  `all`: experts floats of this token.
template <int DT, int L, int VPL>
__device__ __forceinline__ uint32_t open_groups(const RouteParams& p, int64_t row, const float (&value)[VPL], float* all, bool inexact, bool& unclear) {
    const int sub = threadIdx.x % L, first = sub * VPL, size = p.experts / p.groups, lanes = size / VPL;
    float one = -CUDART_INF_F, two = -CUDART_INF_F, second = 0.f;
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
        second = two;
        const int from = min(L - 1, sub * lanes);
        one = __shfl_sync(0xFFFFFFFFu, one, from, L);
        two = __shfl_sync(0xFFFFFFFFu, two, from, L);
    } else {
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            if (first + i < p.experts) all[first + i] = value[i];
        }
        __syncwarp();
        // as many lanes per group as there are, a power of two of them: 17885 x 300 in 4 groups 55 us, with one lane each 71
        int share = 1;
        while (2 * share * p.groups <= L) share *= 2;
        const int group = sub / share;
        if (group < p.groups) {
            for (int i = sub % share; i < size; i += share) {
                const float v = all[group * size + i];
                two = fmaxf(two, fminf(one, v));
                one = fmaxf(one, v);
            }
        }
        __syncwarp();
        for (int o = 1; o < share; o <<= 1) {
            const float a = __shfl_xor_sync(0xFFFFFFFFu, one, o), b = __shfl_xor_sync(0xFFFFFFFFu, two, o);
            two = fmaxf(fminf(one, a), fmaxf(two, b));
            one = fmaxf(one, a);
        }
        const int from = min(L - 1, sub * share);
        one = __shfl_sync(0xFFFFFFFFu, one, from, L);
        two = __shfl_sync(0xFFFFFFFFu, two, from, L);
    }
    const float mine = p.group_top == 2 && two > -CUDART_INF_F ? one + two : one;
    const bool some = sub < p.groups && mine > -CUDART_INF_F;
    uint32_t open = best_groups<L>(p, mine, some);
    if (!inexact) return open;
    // a sum is as good as its parts, which may be larger than it
    const bool in = open >> sub & 1u;
    const float slack = margin(p, fmaxf(fabsf(one), two > -CUDART_INF_F ? fabsf(two) : 0.f));
    const float low = seg_max<L>(in ? slack - mine : -CUDART_INF_F), next = seg_max<L>(some && !in ? mine + slack : -CUDART_INF_F);
    unclear = next > -CUDART_INF_F && !(-low > next);
    if (!in_lanes || !p.sigmoid || !__any_sync(0xFFFFFFFFu, unclear)) return open;
    // the exact scores of the two best of every group: what is not below the second one by more than the error
    double a = -CUDART_INF, b = -CUDART_INF;
    uint32_t close = 0u;
    const float cut = second - margin(p, second);
#pragma unroll
    for (int i = 0; i < VPL; ++i) close |= value[i] > -CUDART_INF_F && !(value[i] < cut) ? 1u << i : 0u;
    while (close != 0u) {
        const int e = first + __ffs(close) - 1;
        close &= close - 1u;
        const double v = exact_sigmoid(load1<DT>(p.logits, row * p.experts + e)) + (p.bias != nullptr ? static_cast<double>(__ldg(p.bias + e)) : 0.0);
        b = v > a ? a : v > b ? v : b;
        a = v > a ? v : a;
    }
    __syncwarp();
    for (int o = 1; o < lanes; o <<= 1) {
        const double c = __shfl_xor_sync(0xFFFFFFFFu, a, o), d = __shfl_xor_sync(0xFFFFFFFFu, b, o);
        b = c > a ? (a > d ? a : d) : (b > c ? b : c);
        a = c > a ? c : a;
    }
    const double sum = p.group_top == 2 && b > -CUDART_INF ? a + b : a;
    open = best_groups<L>(p, __shfl_sync(0xFFFFFFFFu, sum, min(L - 1, sub * lanes), L), some);
    unclear = false;
    return open;
}

template <int L>
constexpr int kRouteRows = 128 / L;  // tokens of a block of four warps

// SCORES: ranks or groups go by scores; otherwise everything goes by logits
template <int DT, int L, int VPL, bool SCORES>
__global__ void __launch_bounds__(128, VPL <= 16 ? 6 : 4) moe_route_kernel(const RouteParams p, int scratch_bytes) {
    extern __shared__ double scratch[];  // scratch_bytes per warp
    constexpr uint32_t kIndex = DT != kDtFp32 ? 0xFFFFu : L * VPL <= 256 ? 0xFFu : 0x3FFu;  // bits of a key that hold the index
    constexpr uint32_t kIndexScore = L * VPL <= 256 ? 0xFFu : 0x3FFu;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % L, seg = lane / L, first = sub * VPL;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRouteRows<L> + warp * (32 / L);
    pdl_wait();
    pdl_release();
    if (row0 >= p.rows) return;
    const bool live = row0 + seg < p.rows;
    const int64_t row = live ? row0 + seg : row0;  // lanes past the last token repeat the first one and keep it to themselves
    double* warp_scratch = reinterpret_cast<double*>(reinterpret_cast<char*>(scratch) + warp * scratch_bytes);
    float x[VPL];
    load_logits<DT, VPL>(p, row, sub, x);
    // a NaN or infinity among the logits, or what a lane lacks of the row: values are looked at one by one then
    float finite = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) finite = fmaf(x[i], 0.f, finite);
    bool odd = __any_sync(0xFFFFFFFFu, finite != 0.f), nan = false;
    if (odd) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) nan |= x[i] != x[i];
        nan = seg_max<L>(nan ? 1.f : 0.f) != 0.f;
    }
    const bool grouped = p.topk_groups < p.groups, by_score = SCORES && p.bias != nullptr;
    constexpr bool need_scores = SCORES;
    float top = 0.f, inv_sum = 0.f;
    if (!p.sigmoid && (need_scores || !p.renormalize)) {
        top = x[0];
#pragma unroll
        for (int i = 1; i < VPL; ++i) top = fmaxf(top, x[i]);
        top = seg_max<L>(top);
        nan = nan || top == CUDART_INF_F;  // a softmax of infinity has no value
        float sum = 0.f;
        if (p.renormalize) {
#pragma unroll
            for (int i = 0; i < VPL; ++i) sum += quick_exp(x[i] - top);
        } else {  // the weights are divided by it: the terms that the backward pass adds
#pragma unroll
            for (int i = 0; i < VPL; ++i) sum += expf(x[i] - top);
        }
        inv_sum = 1.f / seg_sum<L>(sum);
    }
    // what a group's score is made of, and, with a bias, what experts are ranked by; -inf: cannot be chosen
    float value[VPL];
    if (need_scores) {
        float b[VPL];
#pragma unroll
        for (int i = 0; i < VPL; ++i) b[i] = 0.f;
        if (by_score && p.vec_bias) {
            if (first < p.experts) {
#pragma unroll
                for (int i = 0; i < VPL; i += 4) *reinterpret_cast<float4*>(b + i) = __ldg(reinterpret_cast<const float4*>(p.bias + first + i));
            }
        } else if (by_score) {
#pragma unroll
            for (int i = 0; i < VPL; ++i) b[i] = first + i < p.experts ? __ldg(p.bias + first + i) : 0.f;
        }
        finite = 0.f;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            value[i] = (p.sigmoid ? quick_sigmoid(x[i]) : quick_exp(x[i] - top) * inv_sum) + b[i];
            finite = fmaf(value[i], 0.f, finite);
        }
        odd = odd || __any_sync(0xFFFFFFFFu, finite != 0.f);
        if (odd) {
#pragma unroll
            for (int i = 0; i < VPL; ++i) value[i] = x[i] > -CUDART_INF_F && value[i] > -CUDART_INF_F ? value[i] : -CUDART_INF_F;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPL; ++i) value[i] = x[i];
        if (odd) {
#pragma unroll
            for (int i = 0; i < VPL; ++i) value[i] = x[i] > -CUDART_INF_F ? x[i] : -CUDART_INF_F;
        }
    }
    bool unclear = false, unclear_groups = false, closed = false;  // closed: all of this lane's experts are
    uint32_t open = 0xFFFFFFFFu;
    if (grouped) {
        open = open_groups<DT, L, VPL>(p, row, value, reinterpret_cast<float*>(warp_scratch) + seg * p.experts, need_scores, unclear_groups);
        const int size = p.experts / p.groups;
        if (size % VPL == 0) {
            closed = first < p.experts && !(open >> (first / size) & 1u);
        } else {
            int group = first / size, end = (group + 1) * size;  // past the row: groups there are none of
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                if (first + i == end) {
                    ++group;
                    end += size;
                }
                if (first + i < p.experts && !(open >> group & 1u)) value[i] = x[i] = -CUDART_INF_F;
            }
            odd = true;
        }
    }
    uint32_t key[VPL];
    const uint32_t index = by_score ? kIndexScore : kIndex;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const float r = by_score ? value[i] : x[i];
        uint32_t o;
        if (DT == kDtFp16 && !by_score) {
            const uint32_t b = __half_as_ushort(__float2half_rn(r + 0.f));
            o = (b ^ (b & 0x8000u ? 0xFFFFu : 0x8000u)) << 16;
        } else {
            o = ordered(r) & ~index;
        }
        key[i] = o | (index - static_cast<uint32_t>(first + i));
    }
    if (odd) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            if (!((by_score ? value[i] : x[i]) > -CUDART_INF_F)) key[i] = 0u;
        }
    }
    sort_down<VPL>(key);
    // the largest key stays in a register, the others wait in shared memory, with a zero behind them
    uint32_t* list = reinterpret_cast<uint32_t*>(warp_scratch) + lane;
#pragma unroll
    for (int i = 1; i < VPL; ++i) list[32 * i] = key[i];
    list[32 * VPL] = 0u;
    uint32_t head = closed ? 0u : key[0];
    const uint32_t* rest = list + 32;
    const bool exact_keys = DT != kDtFp32 && !by_score;
    const int candidates = exact_keys ? p.k : min(p.k + 1, L), turns = exact_keys ? p.k : candidates + 1;
    uint32_t taken = 0u, next = 0u;
    for (int j = 0; j < turns; ++j) {
        uint32_t m = head;
#pragma unroll
        for (int o = L / 2; o >= 1; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        if (head == m && m != 0u) {
            head = *rest;
            rest += 32;
        }
        if (sub == j) taken = m;
        next = m;
    }
    if (sub >= candidates) taken = 0u;
    int expert = taken != 0u ? static_cast<int>(index - (taken & index)) : -1, where = sub;  // this lane's choice and its place
    float l = expert >= 0 ? load1<DT>(p.logits, row * p.experts + expert) : -CUDART_INF_F;
    if (!exact_keys) {
        const uint32_t kth = __shfl_sync(0xFFFFFFFFu, taken, p.k - 1, L);
        // what was not taken is below `above`
        const uint32_t low = kth & ~index, above = next | index;
        if (next != 0u) unclear = by_score ? !(unordered(low) - unordered(above) > margin(p, unordered(low))) : low <= above;
        int before = 0;
        if (!by_score) {
            const unsigned long long mine = expert >= 0 ? static_cast<unsigned long long>(ordered(l)) << 32 | static_cast<uint32_t>(~expert) : 0ull;
            for (int j = 0; j < candidates; ++j) before += __shfl_sync(0xFFFFFFFFu, mine, j, L) > mine;
        } else {
            double r = -CUDART_INF;
            if (p.sigmoid) {
                r = expert >= 0 ? exact_sigmoid(l) + static_cast<double>(__ldg(p.bias + expert)) : -CUDART_INF;
            } else {
                double sum = 0.0;
#pragma unroll 1
                for (int i = 0; i < VPL; ++i) sum += first + i < p.experts ? exp(static_cast<double>(load1<DT>(p.logits, row * p.experts + first + i)) - static_cast<double>(top)) : 0.0;
#pragma unroll
                for (int o = L / 2; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
                if (expert >= 0) r = exp(static_cast<double>(l) - static_cast<double>(top)) / sum + static_cast<double>(__ldg(p.bias + expert));
            }
            for (int j = 0; j < candidates; ++j) {
                const double o = __shfl_sync(0xFFFFFFFFu, r, j, L);
                const int e = __shfl_sync(0xFFFFFFFFu, expert, j, L);
                before += o > r || (o == r && static_cast<unsigned>(e) < static_cast<unsigned>(expert));
            }
        }
        if (expert >= 0) where = before;
        if (where >= p.k) expert = -1;
    }
    // rows that are not clear, one after the other by all lanes
    uint32_t again = __ballot_sync(0xFFFFFFFFu, live && (unclear || unclear_groups) && sub == 0);
    while (again != 0u) {
        const int from = __ffs(again) - 1;
        again &= again - 1u;
        const int64_t r = __shfl_sync(0xFFFFFFFFu, row, from);
        const bool by_logit = __shfl_sync(0xFFFFFFFFu, !by_score && !unclear_groups, from);
        const uint32_t o = __shfl_sync(0xFFFFFFFFu, open, from);
        __syncwarp();
        const int got = by_logit ? choose_by_logit<DT>(p, r, o, reinterpret_cast<float*>(warp_scratch)) : choose_in_64_bits<DT>(p, r, warp_scratch);
        const int e = __shfl_sync(0xFFFFFFFFu, got, sub);
        if (lane / L == from / L) {
            expert = sub < p.k ? e : -1;
            where = sub;
            l = expert >= 0 ? load1<DT>(p.logits, r * p.experts + expert) : -CUDART_INF_F;
        }
    }
    if (expert < 0) l = -CUDART_INF_F;
    float w;
    if (p.renormalize) {
        // relative to the largest chosen one, so that scores that fp32 cannot hold keep their ratios
        float m = seg_max<L>(l);
        if (p.sigmoid) m = fminf(m, 0.f);
        w = expert < 0 ? 0.f : p.sigmoid ? expf(fminf(l, 0.f) - m) / (1.f + expf(-fabsf(l))) : expf(l - m);
        const float sum = seg_sum<L>(w);
        w = expert < 0 ? 0.f : w / sum;
    } else {
        w = expert < 0 ? 0.f : p.sigmoid ? sigmoidf(l) : expf(l - top) * inv_sum;
    }
    if (live && (expert >= 0 || (where == sub && sub < p.k))) {
        p.idx[row * p.k + where] = expert;
        p.weights[row * p.k + where] = nan ? CUDART_NAN_F : w * p.scale;
    }
}

// The places of load_logits with SPREAD
template <int DT, int VPL>
__device__ __forceinline__ void store_logits(const RouteParams& p, int64_t row, int lane, const float* x) {
    constexpr int kShare = VPL * kBytes<DT>;
    const int64_t at = row * p.experts + lane * VPL;
    if (kShare >= 16 && p.vec) {
        if (lane * VPL >= p.experts) return;
        char* to = static_cast<char*>(p.dlogits) + at * kBytes<DT>;
        if constexpr (DT == kDtFp32 && kShare >= 32) {
#pragma unroll
            for (int i = 0; i < VPL; i += 8) store32(to + i * 4, reinterpret_cast<const uint32_t*>(x + i));
        } else if constexpr (DT == kDtFp32 && kShare == 16) {
            *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(x);
        } else if constexpr (kShare >= 32) {
#pragma unroll
            for (int i = 0; i < VPL; i += 16) {
                const uint4 a = narrow8<DT>(x + i).v[0], b = narrow8<DT>(x + i + 8).v[0];
                const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                store32(to + i * 2, w);
            }
        } else if constexpr (kShare == 16) {
            *reinterpret_cast<uint4*>(to) = narrow8<DT>(x).v[0];
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int e = i * 32 + lane;
            if (e < p.experts) store1<DT>(p.dlogits, row * p.experts + e, x[i]);
        }
    }
}

// One warp per row: all of it without the chosen experts' own terms, then those in their places.
//   renormalised: q = weight / scale, dlogit = scale (dw - sum(dw q)) q, times 1 - score with sigmoid
//   otherwise: softmax scale score (dw - sum(dw score)) over all experts, sigmoid scale dw score (1 - score)
template <int DT, int VPL>
__global__ void __launch_bounds__(256) moe_route_backward_kernel(const RouteParams p) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = p.experts;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + warp;
    pdl_wait();
    pdl_release();
    if (row >= p.rows) return;
    const int64_t row0 = row * e;
    int64_t id64 = lane < p.k ? __ldg(p.idx + row * p.k + lane) : -1;
    const int id = id64 >= 0 && id64 < e ? static_cast<int>(id64) : -1;
    const float g = id >= 0 ? __ldg(p.dweights + row * p.k + lane) * p.scale : 0.f;
    const float l = id >= 0 ? load1<DT>(p.logits, row0 + id) : -CUDART_INF_F;
    float all[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) all[i] = 0.f;
    float d, rest = 0.f;  // gradient of the expert in this place by its own weight, and by those of the others where all experts have one
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
        load_logits<DT, VPL, true>(p, row, lane, all);
        float top = all[0];
#pragma unroll
        for (int i = 1; i < VPL; ++i) top = fmaxf(top, all[i]);
        top = warp_max(top);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < VPL; ++i) sum += all[i] = expf(all[i] - top);
        const float inv_sum = 1.f / warp_sum(sum), q = id >= 0 ? expf(l - top) * inv_sum : 0.f, along = warp_sum(g * q);
        d = g * q;
        rest = -along * q;
        // a row of nothing but -inf has no scores
#pragma unroll
        for (int i = 0; i < VPL; ++i) all[i] = top > -CUDART_INF_F ? -along * all[i] * inv_sum : 0.f;
    }
    // no two places hold one expert, unless the caller made them so: then the first of them takes the sum
    const uint32_t twins = __match_any_sync(0xFFFFFFFFu, id);
    bool lead = id >= 0;
    if (__any_sync(0xFFFFFFFFu, id >= 0 && twins != 1u << lane)) {
        float sum = 0.f;
        for (int j = 0; j < p.k; ++j) {
            const float o = __shfl_sync(0xFFFFFFFFu, d, j);
            if (twins >> j & 1u) sum += o;
        }
        d = sum;
        lead = lead && __ffs(twins) - 1 == lane;
    }
    store_logits<DT, VPL>(p, row, lane, all);
    __syncwarp();
    if (lead) store1<DT>(p.dlogits, row0 + id, d + rest);
}

// Whether a lane's share can be read in pieces of 32 bytes, or one of 16: it is whole ones and so is the row
template <int DT>
bool whole_pieces(const RouteParams& p, int vpl) {
    const int share = vpl * kBytes<DT>;
    if (p.experts % vpl != 0 || share < 16) return false;
    return share >= 32 ? aligned32(p.logits) && aligned32(p.dlogits) && p.experts * kBytes<DT> % 32 == 0
                       : aligned16(p.logits) && aligned16(p.dlogits) && p.experts * kBytes<DT> % 16 == 0;
}

template <int DT, int L, int VPL>
int launch_route(RouteParams p, cudaStream_t stream) {
    p.vec = whole_pieces<DT>(p, VPL);
    p.vec_bias = p.experts % VPL == 0 && aligned16(p.bias);
    // of a warp: a row of doubles, a row of floats for each token, the lanes' lists; one after the other
    const int floats = 32 / L * p.experts * 4, doubles = p.experts * 8, lists = (VPL + 1) * 128;
    int scratch = floats > doubles ? floats : doubles;
    scratch = ((scratch > lists ? scratch : lists) + 15) / 16 * 16;
    const dim3 grid(static_cast<unsigned>((p.rows + kRouteRows<L> - 1) / kRouteRows<L>));
    const bool scores = p.bias != nullptr || (p.topk_groups < p.groups && p.group_top == 2);
    return launch_pdl(scores ? moe_route_kernel<DT, L, VPL, true> : moe_route_kernel<DT, L, VPL, false>, grid, 128, static_cast<size_t>(4) * scratch, stream, p, scratch);
}

template <int DT>
int launch_route_type(const RouteParams& p, cudaStream_t stream) {
    // lanes of a token: as few as hold sixteen experts each, the candidates one each and the groups one each
    int need = (p.experts + 15) / 16;
    const int candidates = DT != kDtFp32 && p.bias == nullptr ? p.k : p.k + 1;
    need = need > candidates ? need : candidates;
    if (p.topk_groups < p.groups && need < p.groups) need = p.groups;
    const int lanes = need <= 8 ? 8 : need <= 16 ? 16 : 32, share = (p.experts + lanes - 1) / lanes;
    if (lanes == 8) return share <= 4 ? launch_route<DT, 8, 4>(p, stream) : share <= 8 ? launch_route<DT, 8, 8>(p, stream) : launch_route<DT, 8, 16>(p, stream);
    if (lanes == 16) return share <= 4 ? launch_route<DT, 16, 4>(p, stream) : share <= 8 ? launch_route<DT, 16, 8>(p, stream) : launch_route<DT, 16, 16>(p, stream);
    if (share <= 4) return launch_route<DT, 32, 4>(p, stream);
    if (share <= 8) return launch_route<DT, 32, 8>(p, stream);
    return share <= 16 ? launch_route<DT, 32, 16>(p, stream) : launch_route<DT, 32, 32>(p, stream);
}

template <int DT, int VPL>
int launch_backward(const RouteParams& p, cudaStream_t stream) {
    return launch_pdl(moe_route_backward_kernel<DT, VPL>, dim3(static_cast<unsigned>((p.rows + 7) / 8)), 256, 0, stream, p);
}

template <int DT>
int launch_backward_type(RouteParams p, cudaStream_t stream) {
    int vpl = 1;
    while (vpl * 32 < p.experts) vpl *= 2;
    p.vec = whole_pieces<DT>(p, vpl);
    switch (vpl) {
        case 1: return launch_backward<DT, 1>(p, stream);
        case 2: return launch_backward<DT, 2>(p, stream);
        case 4: return launch_backward<DT, 4>(p, stream);
        case 8: return launch_backward<DT, 8>(p, stream);
        case 16: return launch_backward<DT, 16>(p, stream);
        default: return launch_backward<DT, 32>(p, stream);
    }
}

template <int DT>
int launch_type(const RouteParams& p, cudaStream_t stream) {
    return p.dlogits != nullptr ? launch_backward_type<DT>(p, stream) : launch_route_type<DT>(p, stream);
}

}  // namespace

}  // namespace cam

// `dlogits` null: the choice and its weights; otherwise the gradient
extern "C" int cam_launch_moe_route(const cam::RouteParams* p, int dtype, cudaStream_t stream) {
    using namespace cam;
    return dtype == kDtBf16 ? launch_type<kDtBf16>(*p, stream) : dtype == kDtFp16 ? launch_type<kDtFp16>(*p, stream) : launch_type<kDtFp32>(*p, stream);
}
