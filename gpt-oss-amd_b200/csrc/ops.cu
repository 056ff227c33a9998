// Host side of the stand-alone operators of include/moe_b200.h: argument checks and launches.
// They need no handle, allocate nothing and keep nothing between calls.
#include <cuda_runtime.h>
#include <float.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>

#include "error.hpp"
#include "op_matvec.cuh"
#include "op_norm.cuh"
#include "op_route.cuh"

using namespace moe::op;

namespace {

constexpr int MAX_DEVICES = 64;
constexpr size_t MV_SM_SMEM = 228 * 1024;  // of an SM

moe_b200_status refuse(moe_b200_status st, const char* fmt, ...) {
    char text[moe::ERROR_BYTES];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof(text), fmt, ap);
    va_end(ap);
    moe::set_thread_error(text);
    return st;
}

#define INVALID(...) return refuse(MOE_B200_ERR_INVALID, __VA_ARGS__)

// A failed CUDA call leaves its error behind, and a later call of the library that asks for the last one would report it.
moe_b200_status cuda_status(const char* what, cudaError_t e) {
    if (e == cudaSuccess)
        return MOE_B200_OK;
    cudaGetLastError();
    return refuse(MOE_B200_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// Device and SM count of the calling thread's current device.
moe_b200_status current_device(int* dev, int* sms) {
    static std::atomic<int> cache[MAX_DEVICES];
    if (cudaGetDevice(dev) != cudaSuccess) {
        cudaGetLastError();
        return refuse(MOE_B200_ERR_NO_DEVICE, "no CUDA device; this library has no CPU path");
    }
    int n = *dev < MAX_DEVICES ? cache[*dev].load(std::memory_order_relaxed) : 0;
    if (n == 0) {
        if (moe_b200_status st = cuda_status("cudaDeviceGetAttribute", cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *dev)))
            return st;
        if (*dev < MAX_DEVICES)
            cache[*dev].store(n, std::memory_order_relaxed);
    }
    *sms = n;
    return MOE_B200_OK;
}

// Launches as a programmatic dependent of the kernel in front (unless pdl_enabled() says no): every kernel here waits for its end before it touches
// global memory, and then lets the next one's blocks come to the SMs (`early`) if it has two blocks per SM at most.
// Behind larger grids they would crowd where room is first: us per call in a replayed chain, launched the ordinary way,
// always early, by this rule: add_rmsnorm 1 x 2880 2.2, 2.0, 2.0; 777 x 2047 6.4, 7.6, 6.3; route_logits 1 x 128 2.7, 2.2,
// 2.2; 3001 x 60 3.6, 3.8, 3.2; w4_matvec 5120 x 2880 6.4, 5.7, 5.7.
template <typename... Params, typename... Args>
cudaError_t launch(void (*kernel)(Params...), unsigned grid, dim3 block, size_t smem, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = moe::pdl_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

bool is_float_type(int dtype) {
    return dtype == MOE_B200_DTYPE_F32 || dtype == MOE_B200_DTYPE_BF16 || dtype == MOE_B200_DTYPE_F16;
}

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// `rows` rows, `stride` elements of `size` bytes apart, on `n`-byte boundaries.
bool rows_aligned(const void* p, int rows, long long stride, int size, size_t n) {
    return aligned(p, n) && (rows <= 1 || ((unsigned long long)stride * (unsigned)size) % n == 0);
}

}  // namespace

extern "C" {

moe_b200_status moe_b200_add_rmsnorm(const moe_b200_add_rmsnorm_args* args, moe_b200_stream stream) {
    if (!args)
        INVALID("moe_b200_add_rmsnorm: null pointer");
    const auto [n_rows, hidden_dim, x, x_dtype, x_stride, residual, residual_dtype, residual_stride, residual_out,
                residual_out_stride, weight, weight_dtype, eps, y, y_dtype, y_stride, q, q_stride, q_scales, q_kind] = *args;
    const int H = hidden_dim;
    if (n_rows < 0 || H <= 0 || H > MOE_B200_ADD_RMSNORM_MAX_HIDDEN)
        INVALID("moe_b200_add_rmsnorm: needs n_rows >= 0 and hidden_dim in 1..%d", MOE_B200_ADD_RMSNORM_MAX_HIDDEN);
    if (!is_float_type(x_dtype) || !is_float_type(weight_dtype) || (residual && !is_float_type(residual_dtype)) ||
        (y && !is_float_type(y_dtype)))
        INVALID("moe_b200_add_rmsnorm: x, residual, weight and y are f32, bf16 or f16");
    if (!(eps >= 0.f && eps <= FLT_MAX))
        INVALID("moe_b200_add_rmsnorm: eps must be finite and not negative");
    int group = 0, mx = 0, n_scales = 1;
    if (q) {
        switch (q_kind) {
            case MOE_B200_SCALE_ROW: break;
            case MOE_B200_SCALE_G32: group = 32; break;
            case MOE_B200_SCALE_G64: group = 64; break;
            case MOE_B200_SCALE_G128: group = 128; break;
            case MOE_B200_SCALE_MX: group = 32, mx = 1; break;
            default: INVALID("moe_b200_add_rmsnorm: unknown scale kind %d", q_kind);
        }
        n_scales = group ? (H + group - 1) / group : 1;
    }
    if (n_rows == 0)
        return MOE_B200_OK;
    if (!y && !q)
        INVALID("moe_b200_add_rmsnorm: neither y nor q asked for");
    if (residual_out && !residual)
        INVALID("moe_b200_add_rmsnorm: residual_out without residual");
    if (!x || !weight || (q && !q_scales))
        INVALID("moe_b200_add_rmsnorm: null pointer");
    if (x_stride < 0 || (residual && residual_stride < 0) || (residual_out && n_rows > 1 && residual_out_stride < H) ||
        (y && n_rows > 1 && y_stride < H) || (q && n_rows > 1 && q_stride < H))
        INVALID("moe_b200_add_rmsnorm: strides of inputs are not negative, rows of outputs do not overlap");
    if (!aligned(x, size_of(x_dtype)) || !aligned(weight, size_of(weight_dtype)) ||
        (residual && !aligned(residual, size_of(residual_dtype))) ||
        (residual_out && !aligned(residual_out, size_of(residual_dtype))) || (y && !aligned(y, size_of(y_dtype))) ||
        (q && !mx && !aligned(q_scales, 4)))
        INVALID("moe_b200_add_rmsnorm: a pointer is not on a boundary of its element type");
    int dev, sms;
    if (moe_b200_status st = current_device(&dev, &sms))
        return st;
    NormArgs a{x, x_stride, x_dtype, residual, residual_out, residual_stride, residual_out_stride, residual_dtype,
               weight, weight_dtype, eps, n_rows, H, y, y_stride, y_dtype, static_cast<uint8_t*>(q), q_stride, q_scales,
               n_scales, group, group == 128 ? 7 : group == 64 ? 6 : 5, mx, 0};
    const bool vec = H % 8 == 0 && rows_aligned(x, n_rows, x_stride, size_of(x_dtype), 16) && aligned(weight, 16) &&
                     (!residual || rows_aligned(residual, n_rows, residual_stride, size_of(residual_dtype), 16)) &&
                     (!residual_out || rows_aligned(residual_out, n_rows, residual_out_stride, size_of(residual_dtype), 16)) &&
                     (!y || rows_aligned(y, n_rows, y_stride, size_of(y_dtype), 16)) && (!q || rows_aligned(q, n_rows, q_stride, 1, 8));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    // Chunks of 256 columns per warp.  Few rows want threads, many rows registers in flight; 1, 2 and 4 chunks, us (bf16,
    // fp32 residual, MX codes): 1 x 2880 2.5, 3.0, 5.1; 256 x 2880 3.6, 3.6, 6.0; 400 x 8192 12.4, 11.1, 14.1; 16384 x 1024 34.7,
    // 35.8, 57.7; 16384 x 2880 97, 95, 146; 5000 x 8192 106, 83, 127.  A block has 32 warps at most, so rows of more than
    // 16384 columns need four, and these do not fit the registers of 1024 threads: up to 800 bytes of a thread go to
    // local memory.  1 x 32768 14.4; 1000 x 32768 114, 66 at the HBM rate.
    const int chunks = (H + 255) / 256;
    const int nv = chunks <= 32 ? (n_rows > 2 * sms && chunks > 4 ? 2 : 1) : chunks <= 64 ? 2 : 4;
    const int threads = 32 * ((chunks + nv - 1) / nv);
    auto kernel = vec ? (nv == 1 ? add_rmsnorm_kernel<true, 1> : nv == 2 ? add_rmsnorm_kernel<true, 2> : add_rmsnorm_kernel<true, 4>)
                      : (nv == 1 ? add_rmsnorm_kernel<false, 1> : nv == 2 ? add_rmsnorm_kernel<false, 2> : add_rmsnorm_kernel<false, 4>);
    const int together = threads == 32 && n_rows >= 8 * sms ? 8 : 1;  // rows per block; 16384 x 64: 5.7 us, one 10.3
    const unsigned grid = (unsigned)(((long long)n_rows + together - 1) / together);
    a.early = grid <= 2u * sms;
    return cuda_status("moe_b200_add_rmsnorm", launch(kernel, grid, dim3(threads, together), 0, st, a));
}

moe_b200_status moe_b200_route_logits(const moe_b200_route_logits_args* args, moe_b200_stream stream) {
    if (!args)
        INVALID("moe_b200_route_logits: null pointer");
    const auto [n_tokens, n_experts, experts_per_token, logits, dtype, stride, score, bias, n_groups, topk_groups, group_top,
                renormalize, scale, topk_i, topk_w, expert_counts] = *args;
    const int E = n_experts, K = experts_per_token;
    if (n_tokens < 0 || n_tokens > MOE_B200_ROUTE_LOGITS_MAX_TOKENS || E <= 0 || E > MOE_B200_ROUTE_LOGITS_MAX_EXPERTS)
        INVALID("moe_b200_route_logits: needs n_tokens in 0..%d and n_experts in 1..%d",
                MOE_B200_ROUTE_LOGITS_MAX_TOKENS, MOE_B200_ROUTE_LOGITS_MAX_EXPERTS);
    if (K <= 0 || K > MOE_B200_ROUTE_LOGITS_MAX_K || K > E)
        INVALID("moe_b200_route_logits: experts_per_token must be in 1..min(%d, n_experts)", MOE_B200_ROUTE_LOGITS_MAX_K);
    if (!is_float_type(dtype))
        INVALID("moe_b200_route_logits: logits are f32, bf16 or f16");
    if (score != MOE_B200_SCORE_SOFTMAX && score != MOE_B200_SCORE_SIGMOID)
        INVALID("moe_b200_route_logits: unknown score %d", score);
    if (n_groups < 1 || n_groups > ROUTE_MAX_GROUPS || E % n_groups || topk_groups < 1 || topk_groups > n_groups)
        INVALID("moe_b200_route_logits: n_groups must be in 1..%d and divide n_experts, topk_groups in 1..n_groups",
                ROUTE_MAX_GROUPS);
    if (n_groups > 1 && (group_top < 1 || group_top > 2 || group_top > E / n_groups))
        INVALID("moe_b200_route_logits: a group is scored by its best or its two best experts");
    if ((long long)topk_groups * (E / n_groups) < K)
        INVALID("moe_b200_route_logits: the groups kept hold fewer than experts_per_token experts");
    if (!(scale >= -FLT_MAX && scale <= FLT_MAX))
        INVALID("moe_b200_route_logits: scale must be finite");
    if (n_tokens > 0 && (!logits || !topk_i || !topk_w))
        INVALID("moe_b200_route_logits: null pointer");
    if (stride < 0)
        INVALID("moe_b200_route_logits: negative stride");
    if (!aligned(logits, size_of(dtype)) || !aligned(bias, 4) || !aligned(topk_i, 4) || !aligned(topk_w, 4) ||
        !aligned(expert_counts, 4))
        INVALID("moe_b200_route_logits: a pointer is not on a boundary of its element type");
    if (n_tokens == 0 && !expert_counts)
        return MOE_B200_OK;
    int dev, sms;
    if (moe_b200_status st = current_device(&dev, &sms))
        return st;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (n_tokens == 0)
        return cuda_status("moe_b200_route_logits: counts", cudaMemsetAsync(expert_counts, 0, sizeof(int) * (size_t)E, st));
    const int nt = E <= 32 ? 1 : E <= 64 ? 2 : E <= 128 ? 4 : E <= 256 ? 8 : 16;
    int lane_shift = 5;
    while (n_groups << lane_shift > 32)
        lane_shift--;
    const bool by_lanes = nt << lane_shift >= E / n_groups;
    LogitsArgs a{logits, stride, dtype, n_tokens, E, K, score == MOE_B200_SCORE_SIGMOID, bias, n_groups, topk_groups,
                 group_top, by_lanes ? lane_shift : 5, by_lanes ? n_groups : 1, by_lanes ? E / n_groups : E, renormalize != 0, scale, topk_i, topk_w, expert_counts, 0};
    const int want = (n_tokens + ROUTE_WARPS - 1) / ROUTE_WARPS, most = 8 * sms;
    const int piece = nt * size_of(dtype) < 16 ? nt * size_of(dtype) : 16;
    const bool vec = a.lane_size % nt == 0 && rows_aligned(logits, n_tokens, stride, size_of(dtype), piece);
    auto kernel = nt == 1 ? (vec ? route_logits_kernel<1, true> : route_logits_kernel<1, false>)
                  : nt == 2 ? (vec ? route_logits_kernel<2, true> : route_logits_kernel<2, false>)
                  : nt == 4 ? (vec ? route_logits_kernel<4, true> : route_logits_kernel<4, false>)
                  : nt == 8 ? (vec ? route_logits_kernel<8, true> : route_logits_kernel<8, false>)
                            : (vec ? route_logits_kernel<16, true> : route_logits_kernel<16, false>);
    const size_t per_warp = nt == 1 ? route_smem_bytes<1>() : nt == 2 ? route_smem_bytes<2>() : nt == 4 ? route_smem_bytes<4>()
                            : nt == 8 ? route_smem_bytes<8>() : route_smem_bytes<16>();
    static_assert(ROUTE_WARPS * (route_smem_bytes<16>() + 128) <= 48 * 1024, "what a block has without asking");
    const int grid = want < most ? want : most;
    a.early = expert_counts || grid <= 2 * sms;  // counts: by a small grid
    cudaError_t e = launch(kernel, grid, 32 * ROUTE_WARPS, per_warp * ROUTE_WARPS, st, a);
    if (e == cudaSuccess && expert_counts) {
        const int n = n_tokens * K, blocks = (n + 2047) / 2048;
        e = launch(route_counts_kernel, blocks < sms ? blocks : sms, 256, 0, st, (const int*)topk_i, n, E, expert_counts);
    }
    return cuda_status("moe_b200_route_logits", e);
}

moe_b200_status moe_b200_w4_matvec(const moe_b200_w4_matvec_args* args, moe_b200_stream stream) {
    if (!args)
        INVALID("moe_b200_w4_matvec: null pointer");
    const auto [matrix, x, x_dtype, x_stride, x_scales, x_scale_kind, n_rows, rows_per_x, ids, swiglu, swiglu_alpha,
                swiglu_limit, out, out_dtype, out_stride] = *args;
    const moe_b200_w4_matrix* w = &matrix;
    const bool int4 = w->format == MOE_B200_W4_INT4;
    if (!int4 && w->format != MOE_B200_W4_MXFP4)
        INVALID("moe_b200_w4_matvec: unknown weight format %d", w->format);
    if (int4 ? (w->group != 32 && w->group != 64 && w->group != 128) : w->group != 32)
        INVALID("moe_b200_w4_matvec: groups of 32 (mxfp4), or 32, 64 or 128 (int4) columns");
    const int N = w->rows, K = w->cols;
    if (N <= 0 || N > MOE_B200_W4_MATVEC_MAX_OUT || K <= 0 || K > MOE_B200_W4_MATVEC_MAX_IN || K % w->group || w->n_mats <= 0)
        INVALID("moe_b200_w4_matvec: needs rows in 1..%d, cols a multiple of the group up to %d, n_mats >= 1",
                MOE_B200_W4_MATVEC_MAX_OUT, MOE_B200_W4_MATVEC_MAX_IN);
    if (n_rows < 0 || n_rows > MOE_B200_W4_MATVEC_MAX_ROWS || rows_per_x <= 0)
        INVALID("moe_b200_w4_matvec: n_rows must be in 0..%d (larger batches are matrix products), rows_per_x >= 1",
                MOE_B200_W4_MATVEC_MAX_ROWS);
    if (!ids && w->n_mats != 1)
        INVALID("moe_b200_w4_matvec: several matrices need ids");
    if (x_dtype != MOE_B200_DTYPE_BF16 && x_dtype != MOE_B200_DTYPE_F16 && x_dtype != MOE_B200_DTYPE_E4M3)
        INVALID("moe_b200_w4_matvec: x is bf16, f16 or e4m3");
    if ((x_dtype == MOE_B200_DTYPE_E4M3) != (x_scale_kind != MOE_B200_SCALE_NONE))
        INVALID("moe_b200_w4_matvec: e4m3 rows need scales, bf16 and f16 rows have none");
    if (!is_float_type(out_dtype))
        INVALID("moe_b200_w4_matvec: out is f32, bf16 or f16");
    if (swiglu && (N % 2 || !(swiglu_limit >= 0.f) || swiglu_alpha != swiglu_alpha))
        INVALID("moe_b200_w4_matvec: SwiGLU needs an even number of rows (gate, up) and a limit");
    int n_xs = 0, xs_shift = 31;
    switch (x_scale_kind) {
        case MOE_B200_SCALE_NONE: break;
        case MOE_B200_SCALE_ROW: n_xs = 1; break;
        case MOE_B200_SCALE_MX:
        case MOE_B200_SCALE_G32: xs_shift = 0; break;
        case MOE_B200_SCALE_G64: xs_shift = 1; break;
        case MOE_B200_SCALE_G128: xs_shift = 2; break;
        default: INVALID("moe_b200_w4_matvec: unknown scale kind %d", x_scale_kind);
    }
    if (xs_shift != 31)
        n_xs = (K + (32 << xs_shift) - 1) / (32 << xs_shift);
    if (n_rows == 0)
        return MOE_B200_OK;
    if (!w->codes || !w->scales || !x || !out || (x_scale_kind != MOE_B200_SCALE_NONE && !x_scales))
        INVALID("moe_b200_w4_matvec: null pointer");
    const int n_out = swiglu ? N / 2 : N;
    if (x_stride < 0 || (n_rows > 1 && out_stride < n_out))
        INVALID("moe_b200_w4_matvec: x_stride is not negative, rows of out do not overlap");
    if (!aligned(w->codes, 16) || !rows_aligned(x, (n_rows - 1) / rows_per_x + 1, x_stride, size_of(x_dtype), x_dtype == MOE_B200_DTYPE_E4M3 ? 8 : 16))
        INVALID("moe_b200_w4_matvec: codes and rows of x must be 16-byte aligned (rows of e4m3 8-byte aligned)");
    if ((int4 && !aligned(w->scales, 2)) || !aligned(w->bias, 4) || !aligned(ids, 4) || !aligned(out, size_of(out_dtype)) ||
        (n_xs && x_scale_kind != MOE_B200_SCALE_MX && !aligned(x_scales, 4)))
        INVALID("moe_b200_w4_matvec: a pointer is not on a boundary of its element type");
    int dev, sms;
    if (moe_b200_status st = current_device(&dev, &sms))
        return st;
    MatvecArgs a{};
    a.codes = w->codes;
    a.scales = w->scales;
    a.bias = w->bias;
    a.n_mats = w->n_mats;
    a.N = N;
    a.K = K;
    a.group_shift = w->group == 128 ? 2 : w->group == 64 ? 1 : 0;
    a.x = x;
    a.x_stride = x_stride;
    a.x_dtype = x_dtype;
    a.x_scales = n_xs ? x_scales : nullptr;
    a.n_xs = n_xs;
    a.xs_shift = xs_shift;
    a.xs_mx = x_scale_kind == MOE_B200_SCALE_MX;
    a.R = n_rows;
    a.rows_per_x = rows_per_x;
    a.ids = ids;
    a.swiglu = swiglu != 0;
    a.alpha = swiglu_alpha;
    a.limit = swiglu_limit;
    a.out = out;
    a.out_stride = out_stride;
    a.out_dtype = out_dtype;
    a.n_tiles = (N + MV_TILE - 1) / MV_TILE;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);

    // Pairs of x rows per pass over the weights.  Chosen matrices are shared by n_rows / n_mats rows on the average.
    // Two pairs halve what is read, but a step has twice the MMAs and the list half the items.  One and two, us:
    // a matrix of its own per row (32 of 2880 x 2880) 29.6, 35.1; four rows per matrix 5.8, 7.3 (2048 x 2880),
    // 8.2, 9.6 (5120), 9.7, 10.2 (8192), 28.7, 25.7 (40224), 14.6, 17.7 (4 x 2880), 25.5, 27.5 (8 x 2880).
    const int share = ids ? (n_rows + w->n_mats - 1) / w->n_mats : n_rows;
    const long long shared_items = (long long)(ids ? w->n_mats : 1) * ((share + 3) / 4) * a.n_tiles;
    int pairs = share <= 2 || shared_items < 5LL * sms ? 1 : 2;
    const int steps = mv_steps(K), sb = int4 ? 2 : 1, SG = (K / 32) >> a.group_shift;
    a.scale_slot = (MV_TILE * SG * sb + 15) / 16 * 16;
    a.scale_bulk = ((reinterpret_cast<uintptr_t>(w->scales) | (ids ? (unsigned long long)N * SG * sb : 0)) & 15) == 0;
    // The ring: rows in as few pieces as leave room for two stages in each of two blocks per SM, or for three in one.
    // Us per 20000 rows, blocks per SM / steps of a piece / stages: 3584 columns 13.4 (2/28/2), 13.6 (2/28/3),
    // 13.6 (1/28/4), 16.6 (2/24/3); 6144 18.9 (1/48/3), 19.8 (1/48/4), 20.9 (2/24/3), 25.2 (1/32/4); 8192 24.8 (1/64/2),
    // 25.4 (2/32/2), 27.6 (1/32/4), 30.6 (2/16/4); 16384 44.3 (1/48/3), 44.2 (1/64/2), 53.4 (2/24/2).  Where x leaves two
    // pairs only short pieces, two passes are faster: 4 rows, two pairs and one: 16384 columns 110 (1/16/3), 98; int4
    // 179 (1/8/4), 118; 12288 int4 73 (1/24/3), 86.
    size_t smem = 0;
    int blocks = 0;
    for (;; pairs /= 2) {
        const size_t fixed = 1024 + mv_static_bytes(pairs);  // the system's and the kernel's own
        const size_t x_bytes = 128 + (size_t)(n_rows < 2 * pairs ? n_rows : 2 * pairs) * steps * 272;
        for (int nc = 1; nc <= (steps + MV_WARPS - 1) / MV_WARPS && !smem; nc++) {
            const int cs = nc == 1 ? steps : ((steps + nc - 1) / nc + MV_WARPS - 1) / MV_WARPS * MV_WARPS;
            if ((steps + cs - 1) / cs != nc)
                continue;
            if (pairs > 1 && nc > 1 && cs < 24)
                break;
            const int pitch = nc == 1 ? K / 2 : cs * 64 + 64;  // pieces of rows 64 modulo 128 apart
            for (blocks = 2; blocks >= 1 && !smem; blocks--)
                for (int d = MV_MAX_DEPTH; d >= (blocks == 2 ? 2 : 3) && !smem; d--) {
                    const int slots = (d - 1 + nc - 1) / nc + 1;  // tiles begun or ahead
                    const size_t need = (size_t)d * MV_TILE * pitch + (size_t)slots * a.scale_slot + x_bytes;
                    if (need <= MV_SM_SMEM / blocks - fixed) {
                        a.depth = d;
                        a.chunk_steps = cs;
                        a.pitch = pitch;
                        a.scale_slots = slots;
                        smem = need;
                    }
                }
        }
        blocks++;
        if (smem || pairs == 1)
            break;
    }
    if (!smem)
        INVALID("moe_b200_w4_matvec: rows too long for shared memory");
    a.row_map = a.pitch % 64 == 32 ? 1 : a.pitch % 32 == 16 ? 2 : 0;
    const bool paired = a.group_shift == 0 && (K / 32) % 2 == 0;
    typedef void (*Kernel)(MatvecArgs);
#define MV_ROW(I4, PR) {w4_matvec_kernel<I4, PR, 1>, w4_matvec_kernel<I4, PR, 2>}
    static const Kernel kernels[2][2][2] = {{MV_ROW(false, false), MV_ROW(false, true)}, {MV_ROW(true, false), MV_ROW(true, true)}};
#undef MV_ROW
    const Kernel kernel = kernels[int4][paired][pairs - 1];
    if (smem > 32 * 1024) {  // with the fixed part more than a block has without asking
        cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)(MV_SM_SMEM - 1024 - mv_static_bytes(pairs)));
        if (e != cudaSuccess)
            return cuda_status("moe_b200_w4_matvec: shared memory", e);
    }
    const long long passes = ids ? n_rows : (n_rows + 2 * pairs - 1) / (2 * pairs);
    const long long items = passes * a.n_tiles, most = (long long)blocks * sms;
    return cuda_status("moe_b200_w4_matvec", launch(kernel, (unsigned)(items < most ? items : most), MV_BLOCK, smem, st, a));
}

}  // extern "C"
