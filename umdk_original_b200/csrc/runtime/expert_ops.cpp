// Host side of the expert-MLP operators that need no Buffer: checks, tensor maps, launches.
#include "expert_ops.h"

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>

#include "../kernels/expert_ops.h"
#include "../kernels/launch.h"
#include "cam_runtime.h"

namespace {

int refuse(const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return cam_fail(buf);
}

#define EXP_CHECK(cond, ...)                     \
    do {                                         \
        if (!(cond)) return refuse(__VA_ARGS__); \
    } while (0)

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// [rows, bytes] with boxes of 128 bytes x box_rows
int map_2d(CUtensorMap* out, const void* base, uint64_t bytes, uint64_t rows, uint32_t box_rows) {
    const uint64_t dims[2] = {bytes, rows}, strides[1] = {bytes};
    const uint32_t box[2] = {128, box_rows};
    return cam_encode_tmap(out, base, 2, dims, strides, box);
}

// [experts, rows, bytes] with boxes of 128 bytes x box_rows
int map_3d(CUtensorMap* out, const void* base, uint64_t bytes, uint64_t rows, uint64_t experts, uint32_t box_rows) {
    const uint64_t dims[3] = {bytes, rows, experts}, strides[2] = {bytes, bytes * rows};
    const uint32_t box[3] = {128, box_rows, 1};
    return cam_encode_tmap(out, base, 3, dims, strides, box);
}

int launched(int rc, const char* what) {
    return rc == 0 ? 0 : refuse("%s: launch failed: %s", what, cudaGetErrorString(static_cast<cudaError_t>(rc)));
}

// A status word per device, in host memory that every device can write: it is there when the call that went wrong has ended, and
// reading it costs the host nothing.  Stays for the life of the process.
constexpr int kMaxDevices = 64;
struct alignas(64) StatusWord {
    CamStatus st;
};
std::atomic<StatusWord*> g_words{nullptr};

StatusWord* status_words() {
    StatusWord* w = g_words.load(std::memory_order_acquire);
    if (w != nullptr) return w;
    static std::mutex lock;
    std::lock_guard<std::mutex> guard(lock);
    w = g_words.load(std::memory_order_relaxed);
    if (w != nullptr) return w;
    void* p = nullptr;
    // the first call may be one that is captured
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    const cudaError_t err = cudaHostAlloc(&p, kMaxDevices * sizeof(StatusWord), cudaHostAllocPortable | cudaHostAllocMapped);
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (err != cudaSuccess) {
        cudaGetLastError();
        return nullptr;
    }
    std::memset(p, 0, kMaxDevices * sizeof(StatusWord));
    g_words.store(static_cast<StatusWord*>(p), std::memory_order_release);
    return static_cast<StatusWord*>(p);
}

// The current device's status word for a product that is about to be launched; refused while an earlier failure stands there.
int status_for_launch(const char* what, CamStatus** out) {
    int dev = 0;
    const cudaError_t err = cudaGetDevice(&dev);
    EXP_CHECK(err == cudaSuccess, "%s: %s", what, cudaGetErrorString(err));
    EXP_CHECK(dev >= 0 && dev < kMaxDevices, "%s: device index %d not supported", what, dev);
    StatusWord* w = status_words();
    EXP_CHECK(w != nullptr, "%s: no host memory for the status word", what);
    CamStatus* st = &w[dev].st;
    const int code = __atomic_load_n(&st->code, __ATOMIC_ACQUIRE);
    EXP_CHECK(code == 0, "%s: an earlier expert product on device %d gave up (%s; who=%d, detail=%d, block=%d) and its results mean nothing; "
              "ops.check_expert_ops() reports and clears this", what, dev, cam_status_string(code), st->who, st->detail, st->block);
    *out = st;
    return 0;
}

// Environment switch: -1 unset, otherwise its number.
int env_switch(const char* name) {
    const char* v = std::getenv(name);
    return v != nullptr && *v != 0 ? std::atoi(v) : -1;
}

// Shape of a product in the form for few rows (expert_gemm_narrow.cu)
struct FewRows {
    int slot_rows, kblocks, chunked, chunks, stages, split;
    int64_t upper;   // row blocks there can be
    int64_t turns, turn_kblocks, turn_fixed;  // turns of the SMs; K-blocks of a tile and cycles beside them in a turn
};

FewRows plan_few_rows(int rows, int num_experts, int64_t n_tiles, int row_bytes, bool fp4) {
    FewRows f{};
    const int sms = cam::sm_count_of_current_device();
    // Room for twice the mean rows per expert: larger experts are cut, and their weights come from L2 for the further tiles.
    const int64_t mean = (static_cast<int64_t>(rows) + num_experts - 1) / num_experts;
    f.slot_rows = rows <= 32 || mean <= 16 ? 32 : rows <= 64 || mean <= 40 ? 64 : 128;
    const int64_t blocks = rows <= num_experts ? rows : static_cast<int64_t>(num_experts) * ((mean + f.slot_rows - 1) / f.slot_rows);
    f.upper = rows / f.slot_rows + (rows < num_experts ? rows : num_experts);
    f.kblocks = (row_bytes + 127) / 128;
    f.chunked = row_bytes % 128 == 0;
    const int per_chunk = (f.slot_rows + 128) * 128, room = 232448 - cam_expert_narrow_fixed_smem(fp4, f.slot_rows);
    f.chunks = f.chunked && f.kblocks > 1 && room / (2 * per_chunk) >= 3 ? 2 : 1;
    const int fit = room / (f.chunks * per_chunk), most = cam_expert_narrow_max_stages();
    f.stages = fit < most ? fit : most;
    // CTAs per tile: turns of the SMs x cycles of a turn (a K-block at an SM's share of the memory bandwidth, a fixed part, the
    // exchange inside the cluster, which the next tile waits for).  Forward pass of one expert of 7168 x 2048 in 16 bits, with 1, 2, 4:
    // 128 rows 62, 52, 52 us (mixed as chosen here 46), 384 rows 77, 81, 118 us.
    const int unit = fp4 ? 4 : f.chunks, units = (f.kblocks + unit - 1) / unit;
    const int forced = env_switch("UMDK_CAM_EXPERT_SPLIT");
    int64_t best = -1;
    for (int split = 1; split <= 4 && split <= units; split *= 2) {  // clusters of 8 find too few places at once
        const int64_t turns = (blocks * n_tiles + sms / split - 1) / (sms / split);
        const int64_t blocks_k = static_cast<int64_t>((units + split - 1) / split) * unit;
        const int64_t fixed = 1500 + (split == 1 ? 0 : turns > 1 ? 2000 * split : fp4 ? 4000 : 2000);
        const int64_t cost = turns * (blocks_k * 770 + fixed);
        if (forced > 0 ? split <= forced : best < 0 || cost < best) {
            best = cost;
            f.split = split;
            f.turns = turns;
            f.turn_kblocks = blocks_k;
            f.turn_fixed = fixed;
        }
    }
    return f;
}

// That form, or CTA pairs?  Up to 128 rows per expert it takes 0.5 - 1.02 of the time of the pairs (1 to 64 experts of 2048 x 768 to
// 7168 x 2048, 16 to 128 rows, 16 and 4 bits).
//
// 4 bits above that: at 160 rows it computes two tiles where the pairs compute one, 1.0 - 1.3.  With fewer than 32 tiles of 256 x 256
// most SMs would stand still in pairs, while this form divides a tile's K-blocks: one expert of 7168 x 2048, 160 - 512 rows, or of 2048 x
// 1024, 160 - 768 rows: 0.75 - 1.15.
bool few_rows_pay_fp4(int rows, int num_experts, int n_dim, bool swiglu) {
    const int sw = env_switch("UMDK_CAM_EXPERT_NARROW");
    if (sw >= 0) return sw != 0;
    const int64_t mean = (static_cast<int64_t>(rows) + num_experts - 1) / num_experts;
    return mean <= 128 || (mean + 255) / 256 * num_experts * ((n_dim + (swiglu ? 127 : 255)) / (swiglu ? 128 : 256)) < 32;
}

// 16 bits, above 128 rows in the forward pass and always in the backward pass: the smaller of two estimates in cycles decides, with
// constants fitted to kernel times (L2 cold) of 66 forward and 44 backward sizes: 1 to 64 experts of 2048 x 768 to 7168 x 2048, 16 to
// 2048 rows each.  A turn of the pairs takes, per K-block, a start and the MMAs of its rows, or the memory's time for the weights if
// many pairs are busy; its tiles are 512 weight rows x 256 rows, with gate and up 256 of each, dact's 256 x 256.
//   forward, pairs / few rows: one expert of 7168 x 2048, 512 rows 105 / 77 us; 8 of 2048 x 1024, 256 rows 60 / 56, 384 rows 56 / 71;
//     4 of 7168 x 2048, 160 rows 103 / 138
//   dact and dx: one of 7168 x 2048, 256 rows 93 / 56, 768 rows 97 / 128; 8 of 2048 x 1024, 128 rows 56 / 50, 384 rows 63 / 87; 16 of
//     4096 x 2048, 375 rows 281 / 425
bool few_rows_pay_16(int rows, int num_experts, int n_dim, int form, int k) {
    const int sw = env_switch("UMDK_CAM_EXPERT_NARROW");
    if (sw >= 0) return sw != 0;
    const bool swiglu = form == cam::kMlpUp, dact = form == cam::kMlpDact, backward = dact || form == cam::kMlpDx;
    const int64_t mean = (static_cast<int64_t>(rows) + num_experts - 1) / num_experts;
    if (!backward && mean <= 128) return true;
    const int step = swiglu ? 64 : 128, wide = swiglu || dact ? 256 : 512;
    const int64_t parts = (mean + 255) / 256, cols = ((mean + parts - 1) / parts + 31) / 32 * 32;
    const int64_t most = cam::sm_count_of_current_device() / 2, live = rows < num_experts ? rows : num_experts;
    const int64_t tiles = live * parts * ((n_dim + wide - 1) / wide), busy = tiles < most ? tiles : most;
    const int64_t turns = (tiles + most - 1) / most, memory = 1420 * busy / most;
    const FewRows f = plan_few_rows(rows, num_experts, (n_dim + step - 1) / step, k * 2, false);
    // tall tiles also take their rows from L2
    const int64_t few = f.turns * (f.turn_kblocks * (dact ? 807 : backward ? 760 : 770 + f.slot_rows) + f.turn_fixed);
    int64_t pairs;
    if (dact) {
        pairs = 4000 + turns * (f.kblocks * (550 + 400 * busy / most) + 1000);
    } else {
        const int64_t work = backward ? 560 + cols * 5 / 2 : 700 + 3 * cols;
        pairs = turns * f.kblocks * (work > memory ? work : memory) + (backward ? 7000 : 18000 * turns);
    }
    return few < pairs;
}

// Up and down of a handful of rows on the ordinary cores (expert_gemv.cu)?  Forward pass, few-row form / this one, steady loop: one
// expert of 7168 x 2048 with 1, 2, 3, 4 rows 26.7 / 19.9, 27.1 / 21.5, 27.3 / 24.4, 26.9 / 27.9 us; 8 of them 28.6 / 21.5, 40 / 36, 58 / 53,
// 64 / 67; 16 of 4096 x 1024 21 / 10, 23 / 16, 26 / 26, 29 / 30.  Small experts gain longer: one of 2048 x 1024, 4 rows 15 / 11, 12 rows
// 16 / 18; 6 of 1000 x 344, 4 - 16 rows 16 - 24 / 10 - 12.
bool gemv_pays(int rows, int n_dim, int k, int form) {
    if (env_switch("UMDK_CAM_EXPERT_NARROW") >= 0 || (form != cam::kMlpUp && form != cam::kMlpDown) || k > cam::kGvMaxSmem / 8) return false;
    return rows <= 3 || (rows <= 16 && static_cast<int64_t>(rows) * n_dim * (form == cam::kMlpUp ? 2 : 1) * k < 1 << 24);
}

// The form for few rows: maps and launch.  `row_bytes` of the row operand (and of the weights' rows, unless they are contracted
// over their rows); n_dim, the operands' scales and outputs are set.
int launch_narrow(cam::NarrowParams* p, int kind, int form, const void* a, const void* w, int row_bytes, const char* what, cudaStream_t stream) {
    const bool swiglu = form == cam::kNarrowSwiglu;
    const int step = swiglu ? 64 : 128;
    const int64_t n_tiles = (p->n_dim + step - 1) / step;
    const FewRows f = plan_few_rows(p->rows, p->num_experts, n_tiles, row_bytes, kind != cam::kNarrow16);
    p->slot_rows = f.slot_rows;
    p->kblocks = f.kblocks;
    p->chunked = f.chunked;
    p->chunks = f.chunks;
    p->stages = f.stages;
    p->stage_bytes = f.chunks * (f.slot_rows + 128) * 128;
    p->split = f.split;
    const uint64_t bytes = p->chunked ? 128 : static_cast<uint64_t>(row_bytes), blocks_k = p->chunked ? static_cast<uint64_t>(p->kblocks) : 1;
    const uint64_t pitch = static_cast<uint64_t>(row_bytes), halves = swiglu ? 2 : 1, n = static_cast<uint64_t>(p->n_dim);
    CUtensorMap ta, tb;
    const uint64_t da[3] = {bytes, static_cast<uint64_t>(p->rows), blocks_k}, sa[2] = {pitch, 128};
    const uint32_t ba[3] = {128, p->chunks > 1 ? static_cast<uint32_t>(p->slot_rows) : 32u, static_cast<uint32_t>(p->chunks)};
    if (cam_encode_tmap(&ta, a, 3, da, sa, ba) != 0) return -1;
    if (form == cam::kNarrowDact || form == cam::kNarrowByRows) {
        if (map_3d(&tb, w, n * 2, static_cast<uint64_t>(row_bytes / 2), static_cast<uint64_t>(p->num_experts), 64) != 0) return -1;
        return launched(cam_launch_expert_gemm_narrow(p, kind, form, f.upper * n_tiles, &ta, &tb, stream), what);
    }
    const uint64_t db[5] = {bytes, n, halves, blocks_k, static_cast<uint64_t>(p->num_experts)}, sb[4] = {pitch, pitch * n, 128, pitch * n * halves};
    const uint32_t bb[5] = {128, static_cast<uint32_t>(step), static_cast<uint32_t>(halves), static_cast<uint32_t>(p->chunks), 1};
    if (cam_encode_tmap(&tb, w, 5, db, sb, bb) != 0) return -1;
    return launched(cam_launch_expert_gemm_narrow(p, kind, form, f.upper * n_tiles, &ta, &tb, stream), what);
}

}  // namespace

extern "C" int cam_quantize_fp4(const void* x, int dtype, int fmt, void* q, void* s, int64_t numel, const float* gscale,
                                int64_t gscales, cudaStream_t stream) {
    if (numel == 0) return 0;
    EXP_CHECK(x && q && s, "quantize_fp4: null operand");
    EXP_CHECK(numel > 0 && numel % (fmt == 0 ? 16 : 32) == 0, "quantize_fp4: %lld values are not whole blocks", static_cast<long long>(numel));
    EXP_CHECK(aligned(x, 32) && aligned(q, 8), "quantize_fp4: x must be 32-byte aligned");
    const int64_t groups = numel / 16;
    EXP_CHECK(gscale == nullptr || (gscales >= 1 && groups % gscales == 0), "quantize_fp4: %lld global scales", static_cast<long long>(gscales));
    return launched(cam_launch_quantize_fp4(x, dtype, fmt, q, s, groups, gscale, gscale && gscales > 1 ? groups / gscales : 0, stream), "quantize_fp4");
}

extern "C" int cam_dequantize_fp4(const void* q, const void* s, int dtype, int fmt, void* out, int64_t numel, const float* gscale,
                                  int64_t gscales, cudaStream_t stream) {
    if (numel == 0) return 0;
    EXP_CHECK(q && s && out, "dequantize_fp4: null operand");
    EXP_CHECK(numel > 0 && numel % (fmt == 0 ? 16 : 32) == 0, "dequantize_fp4: %lld values are not whole blocks", static_cast<long long>(numel));
    EXP_CHECK(aligned(q, 8) && aligned(out, 32), "dequantize_fp4: q must be 8-byte aligned");
    const int64_t groups = numel / 16;
    EXP_CHECK(gscale == nullptr || (gscales >= 1 && groups % gscales == 0), "dequantize_fp4: %lld global scales", static_cast<long long>(gscales));
    return launched(cam_launch_dequantize_fp4(q, s, dtype, fmt, out, groups, gscale, gscale && gscales > 1 ? groups / gscales : 0, stream), "dequantize_fp4");
}

extern "C" int cam_grouped_gemm_fp4(const void* a_q, const void* a_s, int rows, const void* w_q, const void* w_s, const int* offsets,
                                    int num_experts, int n_dim, int k_dim, int fmt, int swiglu, const float* a_gscale,
                                    const float* w_gscale, const float* out_gscale, void* out, void* out_s, cudaStream_t stream) {
    EXP_CHECK(a_q && a_s && w_q && w_s && offsets && out && (!swiglu || out_s), "grouped_gemm_fp4: null operand");
    EXP_CHECK(rows >= 1 && num_experts >= 1, "grouped_gemm_fp4: empty problem");
    EXP_CHECK(k_dim >= 128 && k_dim % 128 == 0, "grouped_gemm_fp4: K %d must be a multiple of 128", k_dim);
    EXP_CHECK(n_dim >= 128 && n_dim % (swiglu ? 256 : 128) == 0, "grouped_gemm_fp4: N %d must be a multiple of %d", n_dim, swiglu ? 256 : 128);
    EXP_CHECK(static_cast<int64_t>(num_experts) * n_dim < (1ll << 31), "grouped_gemm_fp4: weight rows overflow");
    EXP_CHECK(aligned(a_s, 4) && aligned(w_s, 4), "grouped_gemm_fp4: scales must be 4-byte aligned");
    CamStatus* status = nullptr;
    if (status_for_launch("grouped_gemm_fp4", &status) != 0) return -1;
    if (few_rows_pay_fp4(rows, num_experts, swiglu ? n_dim / 2 : n_dim, swiglu != 0)) {
        cam::NarrowParams p{};
        p.status = status;
        p.expert_offsets = offsets;
        p.num_experts = num_experts;
        p.rows = rows;
        p.n_dim = swiglu ? n_dim / 2 : n_dim;
        p.out = out;
        p.a_scales = static_cast<const uint8_t*>(a_s);
        p.b_scales = static_cast<const uint8_t*>(w_s);
        p.scale_pitch = k_dim / (fmt == 0 ? 16 : 32);
        p.scale_vec = k_dim % 256 == 0 && aligned(a_s, 16) && aligned(w_s, 16);
        p.a_gscale = a_gscale;
        p.b_gscale = w_gscale;
        p.out_gscale = out_gscale;
        p.out_scales = static_cast<uint8_t*>(out_s);
        return launch_narrow(&p, fmt, swiglu ? cam::kNarrowSwiglu : cam::kNarrowPlain, a_q, w_q, k_dim / 2, "grouped_gemm_fp4", stream);
    }
    cam::GroupedGemmFp4Params p{};
    p.status = status;
    p.expert_offsets = offsets;
    p.num_experts = num_experts;
    p.rows = rows;
    p.n_dim = n_dim;
    p.k_dim = k_dim;
    p.a_scales = static_cast<const uint8_t*>(a_s);
    p.b_scales = static_cast<const uint8_t*>(w_s);
    p.scale_vec = k_dim % 256 == 0 && aligned(a_s, 16) && aligned(w_s, 16);
    p.a_gscale = a_gscale;
    p.b_gscale = w_gscale;
    p.out_gscale = out_gscale;
    p.out = out;
    p.out_scales = static_cast<uint8_t*>(out_s);
    CUtensorMap ta, ta32, tb, tout;
    const uint64_t bytes = static_cast<uint64_t>(k_dim) / 2;
    if (map_2d(&ta, a_q, bytes, static_cast<uint64_t>(rows), 128) != 0) return -1;
    if (map_2d(&ta32, a_q, bytes, static_cast<uint64_t>(rows), 32) != 0) return -1;
    if (map_2d(&tb, w_q, bytes, static_cast<uint64_t>(num_experts) * n_dim, 128) != 0) return -1;
    if (!swiglu && map_2d(&tout, out, static_cast<uint64_t>(n_dim) * 2, static_cast<uint64_t>(rows), 32) != 0) return -1;
    return launched(cam_launch_grouped_gemm_fp4(&p, fmt, swiglu, &ta, &ta32, &tb, swiglu ? &tb : &tout, stream), "grouped_gemm_fp4");
}

namespace {

// A product of the rows a [rows, k] with the weights: w [E, w_rows, w_cols], contracted over its columns or (by_rows) its rows.
int row_product(int form, const char* what, const void* a, int k, const void* w, int w_rows, int w_cols, bool by_rows, int n,
                const int* offsets, int rows, int num_experts, int dtype, void* out, float* gate_up, cudaStream_t stream) {
    EXP_CHECK(a && w && offsets && out, "%s: null operand", what);
    EXP_CHECK(rows >= 1 && num_experts >= 1, "%s: empty problem", what);
    EXP_CHECK(k >= 8 && n >= 8 && k % 8 == 0 && n % 8 == 0, "%s: sizes %d and %d must be multiples of 8", what, k, n);
    CamStatus* status = nullptr;
    if (status_for_launch(what, &status) != 0) return -1;
    if (gemv_pays(rows, n, k, form)) {
        EXP_CHECK(aligned(a, 16) && aligned(w, 16), "%s: rows and weights must be 16-byte aligned", what);
        cam::GroupedMlpParams p{};
        p.expert_offsets = offsets;
        p.num_experts = num_experts;
        p.rows = rows;
        p.n_dim = n;
        p.k_dim = k;
        p.fp16 = dtype == 1;
        p.out = out;
        p.gate_up = gate_up;
        return launched(cam_launch_expert_gemv(&p, form == cam::kMlpUp, a, w, stream), what);
    }
    if (few_rows_pay_16(rows, num_experts, n, form, k)) {
        cam::NarrowParams p{};
        p.status = status;
        p.expert_offsets = offsets;
        p.num_experts = num_experts;
        p.rows = rows;
        p.n_dim = n;
        p.fp16 = dtype == 1;
        p.out = out;
        p.gate_up = gate_up;
        const int narrow = form == cam::kMlpUp ? cam::kNarrowSwiglu : form == cam::kMlpDact ? cam::kNarrowDact : by_rows ? cam::kNarrowByRows : cam::kNarrowPlain;
        return launch_narrow(&p, cam::kNarrow16, narrow, a, w, k * 2, what, stream);
    }
    cam::GroupedMlpParams p{};
    p.status = status;
    p.expert_offsets = offsets;
    p.num_experts = num_experts;
    p.rows = rows;
    p.n_dim = n;
    p.k_dim = k;
    p.fp16 = dtype == 1;
    p.out = out;
    p.gate_up = gate_up;
    CUtensorMap ta, ta32, tb;
    if (map_2d(&ta, a, static_cast<uint64_t>(k) * 2, static_cast<uint64_t>(rows), 128) != 0) return -1;
    if (map_2d(&ta32, a, static_cast<uint64_t>(k) * 2, static_cast<uint64_t>(rows), 32) != 0) return -1;
    if (map_3d(&tb, w, static_cast<uint64_t>(w_cols) * 2, static_cast<uint64_t>(w_rows), static_cast<uint64_t>(num_experts), by_rows ? 64 : 128) != 0) return -1;
    CUtensorMap tout;
    const uint64_t width = static_cast<uint64_t>(n) * 2;
    if (form == cam::kMlpDact) {
        const uint64_t dims[3] = {width, 2, static_cast<uint64_t>(rows)}, strides[2] = {width, 2 * width};
        const uint32_t box[3] = {128, 1, 32};
        if (cam_encode_tmap(&tout, out, 3, dims, strides, box) != 0) return -1;
    } else if (map_2d(&tout, out, width, static_cast<uint64_t>(rows), 32) != 0) {
        return -1;
    }
    return launched(cam_launch_grouped_mlp(&p, form, &ta, &ta32, &tb, &tout, stream), what);
}

}  // namespace

extern "C" int cam_grouped_mlp_up(const void* x, const void* w1, const int* offsets, int rows, int num_experts, int h, int inter,
                                  int dtype, void* act, float* gate_up, cudaStream_t stream) {
    return row_product(cam::kMlpUp, "grouped_mlp (gate and up)", x, h, w1, 2 * inter, h, false, inter, offsets, rows, num_experts, dtype, act, gate_up, stream);
}

extern "C" int cam_grouped_mlp_down(const void* act, const void* w2, const int* offsets, int rows, int num_experts, int h, int inter,
                                    int dtype, void* y, cudaStream_t stream) {
    return row_product(cam::kMlpDown, "grouped_mlp (down)", act, inter, w2, h, inter, false, h, offsets, rows, num_experts, dtype, y, nullptr, stream);
}

extern "C" int cam_grouped_mlp_dact(const void* dy, const void* w2, const float* gate_up, const int* offsets, int rows, int num_experts,
                                    int h, int inter, int dtype, void* dgu, cudaStream_t stream) {
    EXP_CHECK(gate_up != nullptr, "grouped_mlp (dact): null operand");
    EXP_CHECK(aligned(gate_up, 32), "grouped_mlp (dact): gate_up must be 32-byte aligned");
    return row_product(cam::kMlpDact, "grouped_mlp (dact)", dy, h, w2, h, inter, true, inter, offsets, rows, num_experts, dtype, dgu,
                       const_cast<float*>(gate_up), stream);
}

extern "C" int cam_grouped_mlp_dx(const void* dgu, const void* w1, const int* offsets, int rows, int num_experts, int h, int inter,
                                  int dtype, void* dx, cudaStream_t stream) {
    return row_product(cam::kMlpDx, "grouped_mlp (dx)", dgu, 2 * inter, w1, 2 * inter, h, true, h, offsets, rows, num_experts, dtype, dx, nullptr, stream);
}

extern "C" int cam_grouped_mlp_dw(const void* a, const void* b, const int* offsets, int rows, int num_experts, int m_dim, int n_dim,
                                  int dtype, void* dw, cudaStream_t stream) {
    EXP_CHECK(a && b && offsets && dw, "grouped_mlp (dw): null operand");
    EXP_CHECK(rows >= 1 && num_experts >= 1, "grouped_mlp (dw): empty problem");
    EXP_CHECK(m_dim >= 8 && n_dim >= 8 && m_dim % 8 == 0 && n_dim % 8 == 0, "grouped_mlp (dw): sizes %d and %d must be multiples of 8", m_dim, n_dim);
    CamStatus* status = nullptr;
    if (status_for_launch("grouped_mlp (dw)", &status) != 0) return -1;
    cam::GroupedMlpParams p{};
    p.status = status;
    p.expert_offsets = offsets;
    p.num_experts = num_experts;
    p.rows = rows;
    p.m_dim = m_dim;
    p.n_dim = n_dim;
    p.fp16 = dtype == 1;
    p.out = dw;
    CUtensorMap ta, tb, tout;
    if (map_3d(&tout, dw, static_cast<uint64_t>(n_dim) * 2, static_cast<uint64_t>(m_dim), static_cast<uint64_t>(num_experts), 128) != 0) return -1;
    if (map_2d(&ta, a, static_cast<uint64_t>(m_dim) * 2, static_cast<uint64_t>(rows), 64) != 0) return -1;
    if (map_2d(&tb, b, static_cast<uint64_t>(n_dim) * 2, static_cast<uint64_t>(rows), 64) != 0) return -1;
    return launched(cam_launch_grouped_mlp(&p, cam::kMlpDw, &ta, &ta, &tb, &tout, stream), "grouped_mlp (dw)");
}

extern "C" int cam_expert_ops_status(CamStatus* out, int clear) {
    *out = CamStatus{};
    StatusWord* w = g_words.load(std::memory_order_acquire);
    if (w == nullptr) return 0;  // no product has been launched
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err == cudaSuccess) err = cudaDeviceSynchronize();
    EXP_CHECK(err == cudaSuccess, "expert_ops_status: %s", cudaGetErrorString(err));
    EXP_CHECK(dev >= 0 && dev < kMaxDevices, "expert_ops_status: device index %d not supported", dev);
    if (__atomic_load_n(&w[dev].st.code, __ATOMIC_ACQUIRE) == 0) return 0;
    *out = w[dev].st;
    if (clear) w[dev].st = CamStatus{};
    return 0;
}

extern "C" int cam_expert_ops_set_status(const CamStatus* st) {
    CamStatus* at = nullptr;
    if (status_for_launch("expert_ops_set_status", &at) != 0) return -1;
    *at = *st;
    return 0;
}
