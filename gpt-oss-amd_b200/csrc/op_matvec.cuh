// w4_matvec: y[m, n] = sum_k W[e(m), n, k] x[m / rows_per_x, k] (+ bias), for few rows m and a
// matrix W of 4-bit codes with a scale per group.
//
// Every weight is read once and used for at most a handful of rows, so HBM bounds the operator: N K / 2
// bytes of codes and N K / 32 of scales.  What the SM has to keep up with is the decoding, about 46
// weights per clock at the HBM rate; one conversion instruction per pair of codes and one warp MMA
// (m16n8k16, fp16 in, fp32 accumulators) for 16 rows x 4 groups x 4 columns leave it room.
//
// Layout of a step.  A warp takes 16 rows of W and four groups of 32 columns: lane (g, t) = (lane / 4,
// lane % 4) loads the 16 bytes of group t of row g and of row g + 8, whole 64-byte pieces of a row per
// four lanes, in checkpoint layout and straight into registers.  The lane's codes are its A
// fragments.  The four lanes of a row thus hold four DIFFERENT groups, and their products must not be
// added before each got its scale; so the B fragment is block-diagonal: column t' of B holds the x of
// group t' in the lanes t = t' and zeros in the others, and column t' of the accumulator is the sum over
// group t' alone.  Columns 4..7 serve a second row of x.  Eight MMAs make the step; then the four
// accumulators of a lane are multiplied by their scales (weight scale * x scale) into fp32 sums.  No weight
// goes through shared memory and no lane waits for another.
//
// x is rounded to nothing: bf16 becomes fp16 after the group of 32 was multiplied by the power of two
// that brings its largest value to [2^14, 2^15), which the x scale of the group takes back (exact but for
// values 2^-38 below the group's largest); e4m3 is a subset of fp16.  Code values are exact in
// fp16, so each product is exact and the sums are fp32.
//
// The eight warps of a block split K; their sums meet in shared memory in warp order.  Blocks walk a
// list of (rows of one matrix, 16-row tile) items in contiguous shares, the next step's codes in
// flight while a step is computed.
#pragma once
#include "op_types.cuh"

namespace moe {
namespace op {

constexpr int MV_WARPS = 8;
constexpr int MV_THREADS = 32 * MV_WARPS;
constexpr int MV_TILE = 16;                                   // rows of W per item
constexpr int MV_MAX_ROWS = MOE_B200_W4_MATVEC_MAX_ROWS;      // one thread per row builds the item list
constexpr int MV_UB = 3;                                      // steps (128 columns) in flight per warp
static_assert(MV_MAX_ROWS <= MV_THREADS, "one thread per row");

struct MatvecArgs {
    const uint8_t* codes;   // [n_mats, N, K / 2]
    const void* scales;     // u8 [n_mats, N, K / 32] or bf16 [n_mats, N, K / group]
    const float* bias;      // [n_mats, N] or null
    int n_mats, N, K;
    int group_shift;        // log2(group / 32)
    const void* x;
    long long x_stride;
    int x_dtype;
    const void* x_scales;   // [x rows, n_xs]: f32 or e8m0; null: none
    int n_xs;
    int xs_shift;           // log2(x group / 32); 31: one scale per row
    int xs_mx;
    int R, rows_per_x;
    const int* ids;
    int swiglu;
    float alpha, limit;
    void* out;
    long long out_stride;
    int out_dtype;
    int n_tiles;
};

// Shared memory behind the fixed part: x rows in fp16, then their scales per group of 32.
__host__ __device__ constexpr int mv_steps(int K) { return (K + 127) / 128; }
__host__ __device__ constexpr size_t mv_smem_bytes(int K, int rows) {
    return (size_t)rows * mv_steps(K) * (128 * 2 + 4 * 4);
}

template <bool INT4>
__device__ __forceinline__ void mv_decode(uint32_t w, uint32_t (&o)[4]) {
    if (INT4) {  // code - 8; pairs of columns (0, 4), (1, 5), (2, 6), (3, 7)
        const uint32_t LO = 0x000F000Fu, HI = 0x00F000F0u, MAGIC = 0x64006400u;  // 1024 | code
        const __half2 sub = __floats2half2_rn(-1032.f, -1032.f), sub16 = __floats2half2_rn(-72.f, -72.f);
        const __half2 inv16 = __floats2half2_rn(0.0625f, 0.0625f);
        const uint32_t v = w >> 8;
        const uint32_t b[4] = {(w & LO) | MAGIC, (w & HI) | MAGIC, (v & LO) | MAGIC, (v & HI) | MAGIC};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __half2 h = *reinterpret_cast<const __half2*>(&b[i]);
            const __half2 r = (i & 1) ? __hfma2(h, inv16, sub16) : __hadd2(h, sub);  // 1024 + 16 c -> c - 8
            o[i] = *reinterpret_cast<const uint32_t*>(&r);
        }
    } else {  // pairs of neighbouring columns
        asm("{\n\t.reg .b8 a, b, c, d;\n\t"
            "mov.b32 {a, b, c, d}, %4;\n\t"
            "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
            "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
            "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
            "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
            : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
            : "r"(w));
    }
}

__device__ __forceinline__ void mv_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A weight scale as fp32.  An e8m0 byte means 2^(byte - 127) for EVERY byte, 255 included, as in
// moe_b200_mxfp4_unpack; 2^128 is no fp32 number, so the sums are kept in units of 2: this is
// 2^(byte - 128), bytes 0 and 1 being subnormals, and the epilogue doubles.
template <bool INT4>
__device__ __forceinline__ float mv_scale(uint32_t raw) {
    if (INT4)
        return __uint_as_float(raw << 16);
    return __uint_as_float(raw > 1u ? (raw - 1u) << 23 : 0x00200000u << raw);
}

struct MvStep {  // one step of a lane as loaded: codes of rows g and g + 8, two scales of each
    uint4 lo, hi;
    uint32_t s_lo, s_hi;
};

// The raw scales of groups sg and sg + 1 of a row whose scales start at element `row` (32-column
// groups past G: 0); mxfp4: bytes 0 and 1 of the result, int4: its halves.
template <bool INT4>
__device__ __forceinline__ uint32_t mv_load_scales(const void* scales, long long row, int sg, int G, int shift, bool paired) {
    if (INT4) {
        const uint16_t* p = static_cast<const uint16_t*>(scales) + row;
        if (paired)  // two neighbours on a word boundary
            return *reinterpret_cast<const uint32_t*>(p + sg);
        uint32_t r = p[sg >> shift];
        if (sg + 1 < G)
            r |= (uint32_t)p[(sg + 1) >> shift] << 16;
        return r;
    }
    const uint8_t* p = static_cast<const uint8_t*>(scales) + row;
    if (paired)
        return *reinterpret_cast<const uint16_t*>(p + sg);
    uint32_t r = p[sg];
    if (sg + 1 < G)
        r |= (uint32_t)p[sg + 1] << 8;
    return r;
}

// P pairs of x rows (columns of the MMA) per pass over the weights.
template <bool INT4, int P>
__global__ void __launch_bounds__(MV_THREADS, 2) w4_matvec_kernel(const MatvecArgs a) {
    constexpr int RP = 2 * P;
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ int s_ids[MV_MAX_ROWS];
    __shared__ int s_lead[MV_MAX_ROWS];
    __shared__ int s_rank[MV_MAX_ROWS];
    __shared__ int s_warp_cnt[MV_WARPS];
    __shared__ int s_rows[RP];
    __shared__ float s_red[2][MV_WARPS][MV_TILE][RP];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int steps = mv_steps(a.K), G = a.K >> 5, SG = G >> a.group_shift;
    uint16_t* xs = reinterpret_cast<uint16_t*>(dyn);                                     // [RP][steps * 128] fp16
    float* xsc = reinterpret_cast<float*>(dyn + (size_t)RP * steps * 128 * 2);           // [RP][steps * 4]

    // the list of leaders: rows that open a pass over their matrix
    int n_lead;
    if (a.ids) {
        int id = -1, rank = 0;
        if (tid < a.R) {
            id = a.ids[tid];
            if (id < 0 || id >= a.n_mats)
                id = -1;
            s_ids[tid] = id;
        }
        __syncthreads();
        if (id >= 0)
            for (int j = 0; j < tid; j++)
                rank += s_ids[j] == id;
        const bool lead = id >= 0 && rank % RP == 0;
        const unsigned votes = __ballot_sync(0xffffffffu, lead);
        if (lane == 0)
            s_warp_cnt[warp] = __popc(votes);
        if (tid < a.R)
            s_rank[tid] = id >= 0 ? rank : -1;
        __syncthreads();
        int base = 0;
        n_lead = 0;
        for (int w = 0; w < MV_WARPS; w++) {
            if (w < warp)
                base += s_warp_cnt[w];
            n_lead += s_warp_cnt[w];
        }
        if (lead)
            s_lead[base + __popc(votes & ((1u << lane) - 1u))] = tid;
        __syncthreads();
    } else {
        n_lead = (a.R + RP - 1) / RP;
    }

    const long long total = (long long)n_lead * a.n_tiles;  // fits an int (checked by the host)
    const int i0 = (int)(total * blockIdx.x / gridDim.x), i1 = (int)(total * (blockIdx.x + 1) / gridDim.x);
    const int per_warp = (steps + MV_WARPS - 1) / MV_WARPS;
    const int b0 = min(warp * per_warp, steps), b1 = min(b0 + per_warp, steps);
    const int units = (per_warp + MV_UB - 1) / MV_UB;  // the same for all warps
    // two scales with one load: neighbours in memory, on a boundary of their size together
    const bool paired = a.group_shift == 0 && (G & 1) == 0 &&
                        (reinterpret_cast<uintptr_t>(a.scales) & (INT4 ? 3u : 1u)) == 0;

    auto mat_of = [&](int li) { return a.ids ? s_ids[s_lead[li]] : 0; };
    auto load = [&](MvStep (&u)[MV_UB], int mat, int tile, int unit) {
        const int row = tile * MV_TILE + g;
        const long long r_lo = (long long)mat * a.N + row;
        const bool ok_lo = row < a.N, ok_hi = row + 8 < a.N;
#pragma unroll
        for (int i = 0; i < MV_UB; i++) {
            const int b = b0 + unit * MV_UB + i, grp = b * 4 + t, sg = b * 4 + 2 * (t & 1);
            const uint32_t none = INT4 ? 0x88888888u : 0u;  // codes of zero
            u[i].lo = u[i].hi = make_uint4(none, none, none, none);
            u[i].s_lo = u[i].s_hi = 0;
            if (b < b1 && grp < G) {
                const uint4* c = reinterpret_cast<const uint4*>(a.codes) + r_lo * G + grp;
                if (ok_lo)
                    u[i].lo = __ldcs(c);
                if (ok_hi)
                    u[i].hi = __ldcs(c + 8 * (long long)G);
            }
            if (b < b1 && sg < G) {
                if (ok_lo)
                    u[i].s_lo = mv_load_scales<INT4>(a.scales, r_lo * SG, sg, G, a.group_shift, paired);
                if (ok_hi)
                    u[i].s_hi = mv_load_scales<INT4>(a.scales, (r_lo + 8) * SG, sg, G, a.group_shift, paired);
            }
        }
    };

    int li = i0 / a.n_tiles, tile = i0 % a.n_tiles;
    MvStep cur[MV_UB], nxt[MV_UB];
    if (i0 < i1)
        load(cur, mat_of(li), tile, 0);

    int cnt = 0, cur_lead = -1, buf = 0;
    for (int item = i0; item < i1; item++) {
        const int mat = mat_of(li);
        const int li_next = tile + 1 == a.n_tiles ? li + 1 : li, tile_next = tile + 1 == a.n_tiles ? 0 : tile + 1;
        if (li != cur_lead) {
            // the rows of this pass, their x in fp16 and its scales
            cur_lead = li;
            __syncthreads();  // the previous pass has been computed
            if (a.ids) {
                const int first = s_rank[s_lead[li]], same = s_ids[s_lead[li]];
                const bool in = tid < a.R && s_ids[tid] == same && s_rank[tid] >= first && s_rank[tid] < first + RP;
                if (in)
                    s_rows[s_rank[tid] - first] = tid;
                cnt = __syncthreads_count(in);
            } else {
                cnt = min(RP, a.R - li * RP);
                if (tid < cnt)
                    s_rows[tid] = li * RP + tid;
                __syncthreads();
            }
            const int chunks = steps * 16;  // of 8 columns; four lanes make a group
            for (int i = tid; i < cnt * chunks; i += MV_THREADS) {
                const int c = i / chunks, k8 = i % chunks, grp = k8 >> 2;
                const long long xr = s_rows[c] / a.rows_per_x;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; e++)
                    v[e] = 0.f;
                float sc = 0.f;
                uint32_t h[4] = {0, 0, 0, 0};
                if (grp < G) {
                    sc = 1.f;
                    if (a.x_scales) {
                        const long long at = xr * a.n_xs + (a.xs_shift == 31 ? 0 : grp >> a.xs_shift);
                        sc = a.xs_mx ? e8m0_to_float(static_cast<const uint8_t*>(a.x_scales)[at])
                                     : static_cast<const float*>(a.x_scales)[at];
                    }
                    if (a.x_dtype == MOE_B200_DTYPE_E4M3) {
                        const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.x) + xr * a.x_stride + k8 * 8);
                        const uint32_t w[4] = {q.x & 0xFFFFu, q.x >> 16, q.y & 0xFFFFu, q.y >> 16};
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[e]) : "h"((uint16_t)w[e]));
                    } else {
                        const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + xr * a.x_stride + k8 * 8);
                        h[0] = q.x;
                        h[1] = q.y;
                        h[2] = q.z;
                        h[3] = q.w;
                    }
                }
                if (a.x_dtype == MOE_B200_DTYPE_BF16) {
                    uint32_t m = 0;  // largest magnitude of the group, as bits
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        m = max(m, max((h[e] << 16) & 0x7FFFFFFFu, h[e] & 0x7FFF0000u));
                    const unsigned quad = 0xFu << (lane & 28);
                    m = max(m, __shfl_xor_sync(quad, m, 1));
                    m = max(m, __shfl_xor_sync(quad, m, 2));
                    const uint32_t ex = max(m >> 23, 14u);
                    const float up = __uint_as_float((268u - ex) << 23);  // 2^(141 - ex)
                    sc = grp < G ? __uint_as_float(max((ex - 14u) << 23, 0x00400000u)) : 0.f;
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        h[e] = floats_to_half2(__uint_as_float(h[e] << 16) * up, __uint_as_float(h[e] & 0xFFFF0000u) * up,
                                               MOE_B200_DTYPE_F16);
                }
                if (INT4) {  // the order of mv_decode's pairs
                    const uint32_t p0 = __byte_perm(h[0], h[2], 0x5410), p1 = __byte_perm(h[0], h[2], 0x7632);
                    const uint32_t p2 = __byte_perm(h[1], h[3], 0x5410), p3 = __byte_perm(h[1], h[3], 0x7632);
                    h[0] = p0;
                    h[1] = p1;
                    h[2] = p2;
                    h[3] = p3;
                }
                reinterpret_cast<uint4*>(xs)[c * chunks + k8] = make_uint4(h[0], h[1], h[2], h[3]);
                if ((k8 & 3) == 0)
                    xsc[c * steps * 4 + grp] = sc;
            }
            __syncthreads();
        }

        float acc[P][4];
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int k = 0; k < 4; k++)
                acc[p][k] = 0.f;

        for (int unit = 0; unit < units; unit++) {
            const bool last = unit + 1 == units;
            if (!last)
                load(nxt, mat, tile, unit + 1);
            else if (item + 1 < i1)
                load(nxt, mat_of(li_next), tile_next, 0);
#pragma unroll
            for (int i = 0; i < MV_UB; i++) {
                const int b = b0 + unit * MV_UB + i;
                if (b >= b1)
                    break;
                float d[P][4];
#pragma unroll
                for (int p = 0; p < P; p++)
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        d[p][k] = 0.f;
                const uint32_t w_lo[4] = {cur[i].lo.x, cur[i].lo.y, cur[i].lo.z, cur[i].lo.w};
                const uint32_t w_hi[4] = {cur[i].hi.x, cur[i].hi.y, cur[i].hi.z, cur[i].hi.w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t l[4], h[4];
                    mv_decode<INT4>(w_lo[k], l);
                    mv_decode<INT4>(w_hi[k], h);
#pragma unroll
                    for (int p = 0; p < P; p++) {
                        if (2 * p >= cnt)
                            break;
                        uint4 x = make_uint4(0, 0, 0, 0);
                        const int c = 2 * p + (g >> 2);
                        if ((g & 3) == t && c < cnt)
                            x = reinterpret_cast<const uint4*>(xs)[(c * steps + b) * 16 + t * 4 + k];
                        mv_mma(d[p], l[0], h[0], l[1], h[1], x.x, x.y);
                        mv_mma(d[p], l[2], h[2], l[3], h[3], x.z, x.w);
                    }
                }
                const float sl0 = mv_scale<INT4>(INT4 ? cur[i].s_lo & 0xFFFFu : cur[i].s_lo & 0xFFu);
                const float sl1 = mv_scale<INT4>(INT4 ? cur[i].s_lo >> 16 : cur[i].s_lo >> 8);
                const float sh0 = mv_scale<INT4>(INT4 ? cur[i].s_hi & 0xFFFFu : cur[i].s_hi & 0xFFu);
                const float sh1 = mv_scale<INT4>(INT4 ? cur[i].s_hi >> 16 : cur[i].s_hi >> 8);
#pragma unroll
                for (int p = 0; p < P; p++) {
                    const int c = 2 * p + (t >> 1);
                    if (c < cnt) {  // the product with the x scale first: the two scales alone may leave fp32
                        const float2 sx = *reinterpret_cast<const float2*>(xsc + (c * steps + b) * 4 + 2 * (t & 1));
                        acc[p][0] = fmaf(d[p][0] * sx.x, sl0, acc[p][0]);
                        acc[p][1] = fmaf(d[p][1] * sx.y, sl1, acc[p][1]);
                        acc[p][2] = fmaf(d[p][2] * sx.x, sh0, acc[p][2]);
                        acc[p][3] = fmaf(d[p][3] * sx.y, sh1, acc[p][3]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < MV_UB; i++)
                cur[i] = nxt[i];
        }

        // rows g and g + 8 of x row 2 p + t / 2: the other two groups are with the neighbouring lane
#pragma unroll
        for (int p = 0; p < P; p++) {
            float lo = acc[p][0] + acc[p][1], hi = acc[p][2] + acc[p][3];
            lo += __shfl_xor_sync(0xffffffffu, lo, 1);
            hi += __shfl_xor_sync(0xffffffffu, hi, 1);
            if ((t & 1) == 0) {
                s_red[buf][warp][g][2 * p + (t >> 1)] = lo;
                s_red[buf][warp][g + 8][2 * p + (t >> 1)] = hi;
            }
        }
        __syncthreads();
        if (warp < P) {  // 16 rows x 2 rows of x per warp
            const int r = tid & 15, c = tid >> 4, n = tile * MV_TILE + r;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < MV_WARPS; w++)
                v += s_red[buf][w][r][c];
            if (!INT4)
                v *= 2.f;  // mv_scale
            if (a.bias && n < a.N)
                v += a.bias[(long long)mat * a.N + n];
            const float up = __shfl_down_sync(0xffffffffu, v, 1);
            if (c < cnt && n < a.N) {
                const long long row = (long long)s_rows[c] * a.out_stride;
                if (!a.swiglu) {
                    store_from_float(a.out, row + n, a.out_dtype, v);
                } else if ((r & 1) == 0) {
                    const float gt = fminf(v, a.limit), u = fminf(fmaxf(up, -a.limit), a.limit);
                    store_from_float(a.out, row + (n >> 1), a.out_dtype, gt / (1.f + expf(-a.alpha * gt)) * (u + 1.f));
                }
            }
        }
        buf ^= 1;
        li = li_next;
        tile = tile_next;
    }

    // rows without a matrix
    if (a.ids) {
        const int n_out = a.swiglu ? a.N >> 1 : a.N;
        for (int m = 0; m < a.R; m++)
            if (s_ids[m] < 0)
                for (long long n = (long long)blockIdx.x * MV_THREADS + tid; n < n_out; n += (long long)gridDim.x * MV_THREADS)
                    store_from_float(a.out, m * a.out_stride + n, a.out_dtype, 0.f);
    }
}

}  // namespace op
}  // namespace moe
