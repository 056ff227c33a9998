// w4_matvec: y[m, n] = sum_k W[e(m), n, k] x[m / rows_per_x, k] (+ bias), for few rows m and a
// matrix W of 4-bit codes with a scale per group.
//
// Every weight is read once and used for at most a handful of rows, so HBM bounds the operator: N K / 2
// bytes of codes and N K / 32 of scales.  What the SM has to keep up with is the decoding, about 46
// weights per clock at the HBM rate: one conversion instruction per pair of codes, and one warp MMA
// (m16n8k16, fp16 in, fp32 accumulators) for 16 rows x 4 groups x 4 columns.
//
// A step.  A warp takes 16 rows of W and four groups of 32 columns: lane (g, t) = (lane / 4, lane % 4)
// has the 16 bytes of group t of a row g and of a row g + 8, in checkpoint layout, and its codes are its A
// fragments as they are.  The four lanes of a row thus hold four DIFFERENT groups, and their products
// must not be added before each got its scale; so the B fragment is block-diagonal: column t' of B
// holds the x of group t' in the lanes t = t' and zeros in the others, and column t' of the accumulator
// is the sum over group t' alone.  Columns 4..7 serve a second row of x.  Eight MMAs make the step; then
// the four accumulators of a lane are multiplied by x scale and weight scale into fp32 sums.
//
// x is rounded to nothing: bf16 becomes fp16 after the group of 32 was multiplied by the power of two
// that brings its largest value to [2^14, 2^15), which the x scale of the group takes back; e4m3 is a subset of
// fp16.  Code values are exact in fp16, so each product is exact and the sums are fp32.
// What does not fit is "far" and stays out of the MMA: in bf16, values more than 2^31 below their group's largest
// (the 8 bits of the others end at 2^-24 or above, where fp16's do), and whole groups whose x scale is not within
// 2^-100..2^103: the products of a group are multiples of 2^-25 and sum to less than 2^24, so with a scale inside
// they stay exact, and finite, before the weight scale joins.  The warps add what is far at the end of a tile, in 64 bits.
//
// The stream.  A ninth warp feeds a ring of up to four stages in shared memory with bulk copies: one
// copy for the codes of a tile of 16 rows, which lie together, and one for its scales; the eight others take the
// steps w, w + 8, ... of every row, so the order of a row's sums depends on nothing but K, and leave their
// sums in shared memory, where the ninth warp adds them in warp order and stores the tile.  Two blocks per SM
// have about 150 KB on the way.  Blocks walk a list of (rows of one matrix, tile) items in contiguous
// shares.
//
// Measured (201088 x 2880, mxfp4, one row: 308 MB, 48 us at the HBM rate).  Loads into registers, 8 rows x 64
// bytes per instruction: 82 us with 32 warps per SM; a ring per warp filled by cp.async in the same
// pattern: 72; a bulk copy per row: 81; one bulk copy per tile: 62.  Now 134 instructions per warp and step
// (56 of them decoding) at 2.3 per clock pace it: 59 clocks per step and SM against 44 at the HBM rate.  int4
// decodes in 9 operations per 8 codes instead of 7: 81 us; a second pair of x rows adds 8 MMAs and
// their x to a step: 85 us for three rows in mxfp4, 101 in int4.  Four pairs per pass were slower than two passes (230 us
// against 164).
#pragma once
#include "common.cuh"
#include "op_types.cuh"
#include "tc5_ptx.cuh"

#include <cuda_fp8.h>

namespace moe {
namespace op {

constexpr int MV_WARPS = 8;
constexpr int MV_THREADS = 32 * MV_WARPS;
constexpr int MV_TILE = 16;                                // rows of W per item
constexpr int MV_MAX_ROWS = MOE_B200_W4_MATVEC_MAX_ROWS;  // one thread per row builds the item list
constexpr int MV_BLOCK = MV_THREADS + 32;                  // the warps that compute, and one that feeds them and stores
constexpr int MV_MAX_DEPTH = 4;                            // stages
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
    // the ring: `depth` stages of 16 row pieces of chunk_steps * 128 columns, `pitch` bytes apart, and scale_slots
    // slots of scale_slot bytes for the scales of a tile
    int depth, chunk_steps, pitch, scale_slots, scale_slot;
    int scale_bulk;         // the scales of a tile begin on a 16-byte boundary
    int row_map;            // which rows lie side by side in shared memory's banks: g and g + 1, + 2 (1) or + 4 (2)
};

// No less than the static shared memory of the kernel.
__host__ __device__ constexpr size_t mv_static_bytes(int P) { return 4096 + MV_MAX_DEPTH * MV_WARPS * 128 * P; }
__host__ __device__ constexpr int mv_steps(int K) { return (K + 127) / 128; }

template <bool INT4>
__device__ __forceinline__ void mv_decode(uint32_t w, uint32_t (&o)[4]) {
    if (INT4) {  // code - 8; pairs of columns (0, 4), (1, 5), (2, 6), (3, 7)
        // 1024 | code, and 1024 + 16 code in the upper nibbles, as is widely done: four bits put into the last ones of
        // fp16's 1024 are added to it.  One three-input operation each, the 1024 kept in a register.
        uint32_t magic;
        asm("mov.b32 %0, 0x64006400;" : "=r"(magic));
        const __half2 sub = __floats2half2_rn(-1032.f, -1032.f), sub16 = __floats2half2_rn(-72.f, -72.f);
        const __half2 inv16 = __floats2half2_rn(0.0625f, 0.0625f);
        const uint32_t v = w >> 8;
        uint32_t b[4];
        asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(b[0]) : "r"(w), "r"(magic));
        asm("lop3.b32 %0, %1, 0x00F000F0, %2, 0xEA;" : "=r"(b[1]) : "r"(w), "r"(magic));
        asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(b[2]) : "r"(v), "r"(magic));
        asm("lop3.b32 %0, %1, 0x00F000F0, %2, 0xEA;" : "=r"(b[3]) : "r"(v), "r"(magic));
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

// c = a b, and c += a b.
__device__ __forceinline__ void mv_mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mv_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two weight scales as fp32, from the low 16 bits (mxfp4: two bytes) or the 32 bits (int4) of `raw`.
template <bool INT4>
__device__ __forceinline__ float2 mv_scales(uint32_t raw) {
    if (!INT4)  // e8m0 -> bf16: 2^(byte - 127), byte 0 a subnormal, byte 255 NaN
        asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(raw) : "h"((uint16_t)raw));
    return make_float2(__uint_as_float(raw << 16), __uint_as_float(raw & 0xFFFF0000u));
}

// The raw scales of groups sg and sg + 1 (sg even) of a row, zeros past the row's G groups; mxfp4: bytes 0 and
// 1 of the result, int4: its halves.  PAIRED: one load, neighbours on a boundary of their size together.
template <bool INT4, bool PAIRED>
__device__ __forceinline__ uint32_t mv_load_scales(const uint8_t* row, int sg, int G, int shift) {
    uint32_t r = 0;
    if (sg < G) {
        if (INT4) {
            const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
            if (PAIRED)
                return *reinterpret_cast<const uint32_t*>(p + sg);
            r = p[sg >> shift];
            if (shift)
                r *= 0x10001u;  // one scale for both
            else if (sg + 1 < G)
                r |= (uint32_t)p[sg + 1] << 16;
        } else {
            if (PAIRED)
                return *reinterpret_cast<const uint16_t*>(row + sg);
            r = row[sg];
            if (sg + 1 < G)
                r |= (uint32_t)row[sg + 1] << 8;
        }
    }
    return r;
}

// Keeps what is computed from `v` where it stands: code that runs seldom would else have its constants computed in
// front of the loops around it, and kept in registers through them.
__device__ __forceinline__ void mv_opaque(int& v) { asm volatile("" : "+r"(v)); }

// The x scale of a group, for rows that have some.
__device__ __forceinline__ float mv_x_scale(const MatvecArgs& a, long long xr, int grp) {
    const long long at = xr * a.n_xs + (a.xs_shift == 31 ? 0 : grp >> a.xs_shift);
    return a.xs_mx ? e8m0_to_float(static_cast<const uint8_t*>(a.x_scales)[at]) : static_cast<const float*>(a.x_scales)[at];
}

// Maxima of two 16-bit lanes.
__device__ __forceinline__ uint32_t mv_max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Magnitudes of a group of bf16, eight values in each lane of a quad: the largest in the low half of the result, 2^16
// less the smallest but zero in the high half (0: all are), so that both are maxima.
__device__ __forceinline__ uint32_t mv_span(const uint32_t (&h)[4], int tid) {
    uint32_t most = 0, least = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const uint32_t v = h[e] & 0x7FFF7FFFu;
        most = mv_max2(most, v);
        least = mv_max2(least, (0x80008000u - v) ^ 0x80008000u);  // 0 stays 0
    }
    most = mv_max2(__byte_perm(most, least, 0x5410), __byte_perm(most, least, 0x7632));
    const unsigned quad = 0xFu << (tid & 28);
    most = mv_max2(most, __shfl_xor_sync(quad, most, 1));
    return mv_max2(most, __shfl_xor_sync(quad, most, 2));
}

// What is far.  A group of bf16 by the exponent field of its largest value, which gives the x scale 2^(field - 141); a value
// of a group that is not; a group of e4m3.
__device__ __forceinline__ uint32_t mv_top(uint32_t span) { return (span & 0xFFFFu) >> 7; }
__device__ __forceinline__ bool mv_far_group(uint32_t span) { return (span & 0xFFFFu) != 0 && mv_top(span) - 41u > 244u - 41u; }
__device__ __forceinline__ bool mv_far_value(uint32_t bits16, uint32_t span) {
    const uint32_t v = bits16 & 0x7FFFu;
    return v != 0 && (v >> 7) + 31u < mv_top(span);
}
__device__ __forceinline__ bool mv_far_scale(float sc) { return !(sc == 0.f || (fabsf(sc) >= 0x1p-100f && fabsf(sc) <= 0x1p103f)); }

// One row of x in fp16 and the scale of each of its groups, by all threads of the block.  Returns whether this thread
// saw something far.
template <bool INT4>
__device__ __forceinline__ bool mv_load_x(const MatvecArgs& a, long long xr, int steps, int G, uint4* xs, float* xsc) {
    bool any = false;
    int tid = threadIdx.x;
    mv_opaque(tid);
    for (int k8 = tid; k8 < steps * 16; k8 += MV_THREADS) {  // eight columns; four lanes make a group
        const int grp = k8 >> 2;
        float sc = 0.f;
        uint32_t h[4] = {0, 0, 0, 0};
        bool is_far = false;
        if (grp < G) {
            sc = a.x_scales ? mv_x_scale(a, xr, grp) : 1.f;
            if (a.x_dtype == MOE_B200_DTYPE_E4M3) {
                const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.x) + xr * a.x_stride + k8 * 8);
                const uint32_t w[4] = {q.x & 0xFFFFu, q.x >> 16, q.y & 0xFFFFu, q.y >> 16};
#pragma unroll
                for (int e = 0; e < 4; e++)
                    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[e]) : "h"((uint16_t)w[e]));
                is_far = mv_far_scale(sc);
                if (is_far) {
                    h[0] = h[1] = h[2] = h[3] = 0;
                    sc = 0.f;
                }
            } else {
                const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + xr * a.x_stride + k8 * 8);
                h[0] = q.x;
                h[1] = q.y;
                h[2] = q.z;
                h[3] = q.w;
            }
        }
        if (a.x_dtype == MOE_B200_DTYPE_BF16) {
            const uint32_t span = mv_span(h, tid);
            uint32_t ex = mv_top(span);
            // a group to look at: the largest value is out of range or zero, or 31 * 128 codes and more above the smallest
            if (ex - 41u > 244u - 41u || (span & 0xFFFFu) + (span >> 16) > 0x10000u + 31u * 128u) {
                if (ex - 41u > 244u - 41u) {
                    is_far = mv_far_group(span);
                    h[0] = h[1] = h[2] = h[3] = 0;
                    ex = 127;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const bool lo = mv_far_value(h[e], span), hi = mv_far_value(h[e] >> 16, span);
                        h[e] &= (lo ? 0u : 0x0000FFFFu) | (hi ? 0u : 0xFFFF0000u);
                        is_far = is_far || lo || hi;
                    }
                }
            }
            const float up = __uint_as_float((268u - ex) << 23);  // 2^(141 - ex)
            sc = __uint_as_float((ex - 14u) << 23);
#pragma unroll
            for (int e = 0; e < 4; e++)
                h[e] = floats_to_half2(__uint_as_float(h[e] << 16) * up, __uint_as_float(h[e] & 0xFFFF0000u) * up, MOE_B200_DTYPE_F16);
        }
        if (INT4) {  // the order of mv_decode's pairs
            const uint32_t p0 = __byte_perm(h[0], h[2], 0x5410), p1 = __byte_perm(h[0], h[2], 0x7632);
            const uint32_t p2 = __byte_perm(h[1], h[3], 0x5410), p3 = __byte_perm(h[1], h[3], 0x7632);
            h[0] = p0;
            h[1] = p1;
            h[2] = p2;
            h[3] = p3;
        }
        xs[k8] = make_uint4(h[0], h[1], h[2], h[3]);
        if ((k8 & 3) == 0)
            xsc[grp] = sc;
        any |= is_far;
    }
    return any;
}

// Groups of this warp's steps w, w + 8, ... of a row of x in which something is far: bit 4 i + j is group j of its i-th step.
__device__ __forceinline__ unsigned long long mv_far_groups(const MatvecArgs& a, long long xr) {
    static_assert(MOE_B200_W4_MATVEC_MAX_IN <= 16 * MV_WARPS * 128, "16 steps of 4 groups in 64 bits");
    const int lane = threadIdx.x & 31;
    unsigned long long all = 0;
#pragma unroll 1
    for (int b = threadIdx.x >> 5, at = 0; b < mv_steps(a.K); b += 2 * MV_WARPS, at += 8) {  // two steps: a group per quad
        const int grp = (b + (lane >> 4) * MV_WARPS) * 4 + (lane >> 2 & 3);
        uint32_t h[4] = {0, 0, 0, 0};
        bool far = false;
        if (grp < a.K >> 5) {
            if (a.x_dtype == MOE_B200_DTYPE_BF16) {
                const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + xr * a.x_stride + grp * 32 + (lane & 3) * 8);
                h[0] = v.x, h[1] = v.y, h[2] = v.z, h[3] = v.w;
            } else {
                far = mv_far_scale(mv_x_scale(a, xr, grp));
            }
        }
        const uint32_t span = mv_span(h, lane);
        far = far || mv_far_group(span) || (span != 0 && mv_far_value(0x10000u - (span >> 16), span));
        const unsigned votes = __ballot_sync(0xffffffffu, far);
#pragma unroll
        for (int q = 0; q < 8; q++)
            all |= (unsigned long long)(votes >> (4 * q) & 1) << (at + q);
    }
    return all;
}

// What is far in a row of x, in those groups, times two rows of a matrix, the same for the four lanes of a quad, which
// share the 32 columns of a group.  Codes and scales of the rows from their first group on.
template <bool INT4>
__device__ __forceinline__ float2 mv_far(const MatvecArgs& a, long long xr, unsigned long long groups, const uint8_t* codes0,
                                         const uint8_t* codes1, const uint8_t* scales0, const uint8_t* scales1) {
    const int lane = threadIdx.x & 31, t = lane & 3;
    const bool bf16 = a.x_dtype == MOE_B200_DTYPE_BF16;
    auto weight = [](uint32_t n) {
        if (INT4)
            return (float)((int)n - 8);
        const uint32_t m = n & 7;
        const float v = m < 2 ? 0.5f * m : 0.25f * ((2 + (m & 1)) << (m >> 1));
        return n & 8 ? -v : v;
    };
    auto scale = [&](const uint8_t* row, int grp) {
        return INT4 ? half_to_float(reinterpret_cast<const uint16_t*>(row)[grp >> a.group_shift], MOE_B200_DTYPE_BF16) : e8m0_to_float(row[grp]);
    };
    double lo = 0.0, hi = 0.0;
#pragma unroll 1
    for (; groups; groups &= groups - 1) {
        const int at = __ffsll(groups) - 1, grp = ((int)(threadIdx.x >> 5) + (at >> 2) * MV_WARPS) * 4 + (at & 3);
        const uint32_t w0 = *reinterpret_cast<const uint32_t*>(codes0 + grp * 16 + t * 4);
        const uint32_t w1 = *reinterpret_cast<const uint32_t*>(codes1 + grp * 16 + t * 4);
        const long long col = xr * a.x_stride + grp * 32 + t * 8;
        // columns that are far in any of the four lanes, and what they are of
        uint32_t todo = 0xFF, span = 0;
        if (bf16) {
            const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + col);
            const uint32_t h[4] = {v.x, v.y, v.z, v.w};
            span = mv_span(h, lane);
            if (!mv_far_group(span)) {
                todo = 0;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    todo |= (mv_far_value(h[e], span) ? 1u : 0u) << (2 * e) | (mv_far_value(h[e] >> 16, span) ? 2u : 0u) << (2 * e);
                todo = __reduce_or_sync(0xffffffffu, todo);
            }
        }
        const bool whole = mv_far_group(span);
        double d0 = 0.0, d1 = 0.0;
#pragma unroll 1
        for (; todo; todo &= todo - 1) {
            const int i = __ffs(todo) - 1;
            float x;
            if (bf16) {
                const uint32_t bits = static_cast<const uint16_t*>(a.x)[col + i];
                x = whole || mv_far_value(bits, span) ? __uint_as_float(bits << 16) : 0.f;
            } else {
                __nv_fp8_e4m3 v;
                v.__x = static_cast<const uint8_t*>(a.x)[col + i];
                x = (float)v;
            }
            d0 += (double)weight(w0 >> (4 * i) & 15) * (double)x;
            d1 += (double)weight(w1 >> (4 * i) & 15) * (double)x;
        }
        const double sx = bf16 ? 1.0 : (double)mv_x_scale(a, xr, grp);
        d0 *= sx * (double)scale(scales0, grp), d1 *= sx * (double)scale(scales1, grp);
        d0 += __shfl_xor_sync(0xffffffffu, d0, 1), d1 += __shfl_xor_sync(0xffffffffu, d1, 1);
        lo += d0 + __shfl_xor_sync(0xffffffffu, d0, 2), hi += d1 + __shfl_xor_sync(0xffffffffu, d1, 2);
    }
    return make_float2((float)lo, (float)hi);
}

// Shared memory of the kernel beside the dynamic part.
template <int P>
struct MvShared {
    alignas(8) uint64_t full[MV_MAX_DEPTH], done[MV_MAX_DEPTH];
    float2 red[MV_MAX_DEPTH][MV_WARPS][P][16];
    int ids[MV_MAX_ROWS];
    int lead[MV_MAX_ROWS];
    int rank[MV_MAX_ROWS];
    int rows[2 * P], store_rows[2 * P];
    int abort;
};

// Where the warps that compute are: the tiles of a pass, and the ring.
struct MvRun {
    int li, cnt, tile, tile_end, stage, slot;
    uint32_t parity;
};

// The sums of the tiles of a pass.  FAR: something of its x is far.  Two instances: one with a test at the end of a tile
// took 66 us for the vocabulary (one row, mxfp4), this takes 62; with one far value in x 102, with one in each of its
// 90 groups 560.
template <bool INT4, bool PAIRED, int P, bool FAR>
__device__ __forceinline__ void mv_tiles(const MatvecArgs& a, MvShared<P>& sh, uint8_t* dyn, MvRun& r) {
    using namespace moe::tc5;
    constexpr int RP = 2 * P, SB = INT4 ? 2 : 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int steps = mv_steps(a.K), G = a.K >> 5, SG = G >> a.group_shift, D = a.depth;
    const int stage_bytes = MV_TILE * a.pitch, scales_at = 128 + D * stage_bytes;
    const int xs_at = scales_at + a.scale_slots * a.scale_slot, xsc_at = xs_at + min(RP, a.R) * steps * 256;
    // Lanes g of the MMA take row gr of each half: eight lanes that read shared memory together have two rows, g even
    // and g + 1, and these should lie 64 bytes apart modulo 128.
    const int gr = a.row_map == 1 ? (g & 4) | (g & 1) << 1 | (g >> 1 & 1) : a.row_map == 2 ? (g & 1) << 2 | g >> 1 : g;
    const bool quad_b = (g & 3) == t;  // lanes of the block diagonal of B
    float acc[P][4];
    // One pair of x rows stays in registers, where the lanes off the diagonal hold zeros for good; of several
    // pairs, those lanes read the zeros in shared memory.
    uint4 x1[4];
    int x_at[P], x_step[P], sc_at[P];
#pragma unroll
    for (int k = 0; k < 4; k++)
        x1[k] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int c = 2 * p + (g >> 2), cs = 2 * p + (t >> 1);
        const bool mine = quad_b && c < r.cnt;
        x_at[p] = mine ? xs_at + (c * steps * 16 + t * 4) * 16 : 0;
        x_step[p] = mine ? 256 : 0;
        sc_at[p] = xsc_at + (min(cs, r.cnt - 1) * steps * 4 + 2 * (t & 1)) * 4;
        acc[p][0] = acc[p][1] = acc[p][2] = acc[p][3] = 0.f;
    }
    unsigned long long far[RP];
    if constexpr (FAR)
#pragma unroll 1
        for (int c = 0; c < r.cnt; c++)
            far[c] = mv_far_groups(a, sh.rows[c] / a.rows_per_x);
#pragma unroll 1
    for (; r.tile < r.tile_end; r.tile++) {
        const int scales_row = scales_at + r.slot * a.scale_slot + gr * SG * SB;
        for (int c0 = 0; c0 < steps; c0 += a.chunk_steps) {
            mbar_wait(smem_u32(&sh.full[r.stage]), r.parity, nullptr, 0, &sh.abort);
            // Warp w takes the steps w, w + 8, ... of a row, whatever the chunks: a row's sums have one order.
            const int c1 = min(c0 + a.chunk_steps, steps);
            const int codes_at = 128 + r.stage * stage_bytes + gr * a.pitch + t * 16 - c0 * 64;
            // offsets of the warp's step, moved on by eight steps at a time
            int b = c0 + warp, sg = b * 4 + 2 * (t & 1), code_at = codes_at + b * 64;
            int x_b[P], sc_b[P];
#pragma unroll
            for (int p = 0; p < P; p++) {
                x_b[p] = x_at[p] + x_step[p] * b;
                sc_b[p] = sc_at[p] + 16 * b;
            }
#pragma unroll 1
            for (; b < c1; b += MV_WARPS) {
                const uint4 c_lo = *reinterpret_cast<const uint4*>(dyn + code_at);
                const uint4 c_hi = *reinterpret_cast<const uint4*>(dyn + code_at + 8 * a.pitch);
                const float2 s_lo = mv_scales<INT4>(mv_load_scales<INT4, PAIRED>(dyn + scales_row, sg, G, a.group_shift));
                const float2 s_hi = mv_scales<INT4>(mv_load_scales<INT4, PAIRED>(dyn + scales_row + 8 * SG * SB, sg, G, a.group_shift));
                const uint32_t w_lo[4] = {c_lo.x, c_lo.y, c_lo.z, c_lo.w}, w_hi[4] = {c_hi.x, c_hi.y, c_hi.z, c_hi.w};
                if (P == 1 && x_step[0]) {
                    const uint4* src = reinterpret_cast<const uint4*>(dyn + x_b[0]);
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        x1[k] = src[k];
                }
                float d[P][4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t l[4], u[4];
                    mv_decode<INT4>(w_lo[k], l);
                    mv_decode<INT4>(w_hi[k], u);
#pragma unroll
                    for (int p = 0; p < P; p++) {
                        const uint4 x = P == 1 ? x1[k] : *reinterpret_cast<const uint4*>(dyn + x_b[p] + 16 * k);
                        if (k == 0)
                            mv_mma_first(d[p], l[0], u[0], l[1], u[1], x.x, x.y);
                        else
                            mv_mma(d[p], l[0], u[0], l[1], u[1], x.x, x.y);
                        mv_mma(d[p], l[2], u[2], l[3], u[3], x.z, x.w);
                    }
                }
#pragma unroll
                for (int p = 0; p < P; p++) {
                    // the product with the x scale first: the two scales alone may leave fp32
                    const float2 sx = *reinterpret_cast<const float2*>(dyn + sc_b[p]);
                    acc[p][0] = fmaf(d[p][0] * sx.x, s_lo.x, acc[p][0]);
                    acc[p][1] = fmaf(d[p][1] * sx.y, s_lo.y, acc[p][1]);
                    acc[p][2] = fmaf(d[p][2] * sx.x, s_hi.x, acc[p][2]);
                    acc[p][3] = fmaf(d[p][3] * sx.y, s_hi.y, acc[p][3]);
                    x_b[p] += x_step[p] * MV_WARPS;
                    sc_b[p] += 16 * MV_WARPS;
                }
                code_at += 64 * MV_WARPS;
                sg += 4 * MV_WARPS;
            }
            if (c1 == steps) {
                // this warp's share of the tile: rows g and g + 8 of x row 2 p + t / 2, two groups here, two with lane t ^ 1
#pragma unroll
                for (int p = 0; p < P; p++) {
                    float lo = acc[p][0] + acc[p][1], hi = acc[p][2] + acc[p][3];
                    lo += __shfl_xor_sync(0xffffffffu, lo, 1);
                    hi += __shfl_xor_sync(0xffffffffu, hi, 1);
                    if constexpr (FAR)
#pragma unroll 1
                        for (int c = 2 * p; c < min(2 * p + 2, r.cnt); c++) {
                            if (!far[c])
                                continue;
                            // the stage has whole rows, or their last pieces
                            const int n = r.tile * MV_TILE + gr;
                            const size_t row = (size_t)(a.ids ? sh.ids[sh.lead[r.li]] : 0) * a.N;
                            const uint8_t* codes0 = c0 == 0 ? dyn + 128 + r.stage * stage_bytes + gr * a.pitch : a.codes + (row + min(n, a.N - 1)) * G * 16;
                            const uint8_t* codes1 = c0 == 0 ? codes0 + 8 * a.pitch : a.codes + (row + min(n + 8, a.N - 1)) * G * 16;
                            const float2 f = mv_far<INT4>(a, sh.rows[c] / a.rows_per_x, far[c], codes0, codes1, dyn + scales_row, dyn + scales_row + 8 * SG * SB);
                            if (c == 2 * p + (t >> 1)) {
                                lo += f.x;
                                hi += f.y;
                            }
                        }
                    if ((t & 1) == 0)
                        sh.red[r.stage][warp][p][gr * 2 + (t >> 1)] = make_float2(lo, hi);
                    acc[p][0] = acc[p][1] = acc[p][2] = acc[p][3] = 0.f;
                }
            }
            __syncwarp();  // all lanes have read the stage and left their sums
            if (lane == 0)
                mbar_arrive(smem_u32(&sh.done[r.stage]));
            if (++r.stage == D) {
                r.stage = 0;
                r.parity ^= 1;
            }
        }
        r.slot = r.slot + 1 == a.scale_slots ? 0 : r.slot + 1;
    }
}

// P pairs of x rows (columns of the MMA) per pass over the weights.
template <bool INT4, bool PAIRED, int P>
__global__ void __launch_bounds__(MV_BLOCK, 2) w4_matvec_kernel(const __grid_constant__ MatvecArgs a) {
    using namespace moe::tc5;
    constexpr int RP = 2 * P;
    constexpr int SB = INT4 ? 2 : 1;  // bytes of a scale
    extern __shared__ __align__(128) uint8_t dyn[];
    __shared__ MvShared<P> sh;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int steps = mv_steps(a.K), G = a.K >> 5, SG = G >> a.group_shift, D = a.depth;
    // dynamic shared memory: zeros, the ring of codes, that of scales, x [min(RP, R)][steps * 128] fp16, its scales
    const int stage_bytes = MV_TILE * a.pitch, scales_at = 128 + D * stage_bytes;
    const int xs_at = scales_at + a.scale_slots * a.scale_slot, xsc_at = xs_at + min(RP, a.R) * steps * 256;
    if (tid < 4)
        reinterpret_cast<uint4*>(dyn)[tid] = make_uint4(0, 0, 0, 0);
    if (tid == 0) {
        for (int i = 0; i < D; i++) {
            mbar_init(smem_u32(&sh.full[i]), 1);
            mbar_init(smem_u32(&sh.done[i]), MV_WARPS);
        }
        sh.abort = 0;
        fence_barrier_init();
    }

    pdl_wait();
    pdl_trigger();

    // the list of leaders: rows that open a pass over their matrix
    int n_lead;
    if (a.ids) {
        int id = -1, rank = 0;
        if (tid < a.R) {
            id = a.ids[tid];
            if (id < 0 || id >= a.n_mats)
                id = -1;
            sh.ids[tid] = id;
        }
        __syncthreads();
        if (id >= 0)
            for (int j = 0; j < tid; j++)
                rank += sh.ids[j] == id;
        if (tid < a.R)
            sh.rank[tid] = id >= 0 ? rank : -1;
        __syncthreads();
        n_lead = 0;
        for (int m0 = 0; m0 < a.R; m0 += 32) {  // every warp finds the same
            const int m = m0 + lane;
            const bool lead = m < a.R && sh.rank[m] >= 0 && sh.rank[m] % RP == 0;
            const unsigned votes = __ballot_sync(0xffffffffu, lead);
            if (lead)
                sh.lead[n_lead + __popc(votes & ((1u << lane) - 1u))] = m;
            n_lead += __popc(votes);
        }
    } else {
        n_lead = (a.R + RP - 1) / RP;
    }
    __syncthreads();
    const long long total = (long long)n_lead * a.n_tiles;  // fits an int (checked by the host)
    const int i0 = (int)(total * blockIdx.x / gridDim.x), i1 = (int)(total * (blockIdx.x + 1) / gridDim.x);
    const int li0 = i0 / a.n_tiles, tile0 = i0 - li0 * a.n_tiles;

    if (warp == MV_WARPS) {
        // ---- feeds the ring, and stores the tiles that the others have summed ----
        // A stage is free, and its tile's sums are complete, when the eight warps have arrived on `done`.
        int l_left = i1 - i0, l_li = li0, l_tile = tile0, l_c0 = 0, l_stage = 0, l_slot = 0;
        auto load = [&]() {
            if (l_left <= 0)
                return;
            const size_t row0 = (size_t)(a.ids ? sh.ids[sh.lead[l_li]] : 0) * a.N + l_tile * MV_TILE;
            const int rows = min(MV_TILE, a.N - l_tile * MV_TILE);
            const int pieces = min(a.chunk_steps * 4, G - l_c0 * 4);  // of 16 bytes
            const uint32_t full = smem_u32(&sh.full[l_stage]);
            const uint8_t* s = static_cast<const uint8_t*>(a.scales) + row0 * SG * SB;
            const int scales = l_c0 == 0 ? rows * SG * SB : 0, bulk = a.scale_bulk ? scales & ~15 : 0;
            const int to = scales_at + l_slot * a.scale_slot;
            if (bulk < scales) {  // what no bulk copy may take; a later tile's may be written over it, after these stores
                for (int i = bulk + lane; i < scales; i += 32)
                    dyn[to + i] = s[i];
                fence_proxy_async_smem();
            }
            __syncwarp();
            if (lane == 0)
                mbar_expect_tx(full, rows * pieces * 16 + bulk);
            __syncwarp();
            if (a.chunk_steps == steps) {  // whole rows, as they lie
                if (lane == 0)
                    bulk_load(smem_u32(dyn) + 128 + l_stage * stage_bytes, a.codes + row0 * G * 16, rows * G * 16, full);
            } else if (lane < rows)
                bulk_load(smem_u32(dyn) + 128 + l_stage * stage_bytes + lane * a.pitch,
                          a.codes + ((row0 + lane) * G + l_c0 * 4) * 16, pieces * 16, full);
            if (lane == 31 && bulk)
                bulk_load(smem_u32(dyn) + to, s, bulk, full);
            l_stage = l_stage + 1 == D ? 0 : l_stage + 1;
            l_c0 += a.chunk_steps;
            if (l_c0 >= steps) {
                l_c0 = 0;
                l_left--;
                l_slot = l_slot + 1 == a.scale_slots ? 0 : l_slot + 1;
                if (++l_tile == a.n_tiles) {
                    l_tile = 0;
                    l_li++;
                }
            }
        };
        for (int i = 0; i < D; i++)
            load();
        int li = li0, tile = tile0, stage = 0, cur_lead = -1, cnt = 0, mat = 0;
        uint32_t parity = 0;
        bool ok = true;
        for (int item = i0; item < i1; item++) {
            if (li != cur_lead) {  // the rows of this pass
                cur_lead = li;
                __syncwarp();
                if (a.ids) {
                    const int first = sh.rank[sh.lead[li]];
                    mat = sh.ids[sh.lead[li]];
                    cnt = 0;
                    for (int m0 = 0; m0 < a.R; m0 += 32) {
                        const int m = m0 + lane;
                        const bool in = m < a.R && sh.ids[m] == mat && sh.rank[m] >= first && sh.rank[m] < first + RP;
                        if (in)
                            sh.store_rows[sh.rank[m] - first] = m;
                        cnt += __popc(__ballot_sync(0xffffffffu, in));
                    }
                } else {
                    cnt = min(RP, a.R - li * RP);
                    if (lane < cnt)
                        sh.store_rows[lane] = li * RP + lane;
                }
                __syncwarp();
            }
            float bias[2];
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const int n = tile * MV_TILE + g + 8 * half;
                bias[half] = a.bias && n < a.N ? a.bias[(size_t)mat * a.N + n] : 0.f;
            }
            float2 v[P];
            for (int c0 = 0; c0 < steps; c0 += a.chunk_steps) {
                ok = ok && mbar_wait(smem_u32(&sh.done[stage]), parity, nullptr, 0, &sh.abort) &&
                     *(volatile int*)&sh.abort == 0;
                ok = __all_sync(0xffffffffu, ok);
                if (c0 + a.chunk_steps >= steps) {
                    // lane: row g of both halves, x row 2 p + t / 2 (the same in lanes t and t ^ 1); warps in order
#pragma unroll
                    for (int p = 0; p < P; p++) {
                        v[p] = make_float2(0.f, 0.f);
#pragma unroll
                        for (int w = 0; w < MV_WARPS; w++) {
                            const float2 r = sh.red[stage][w][p][lane >> 1];
                            v[p].x += r.x;
                            v[p].y += r.y;
                        }
                    }
                    __syncwarp();
                }
                if (ok)
                    load();
                if (++stage == D) {
                    stage = 0;
                    parity ^= 1;
                }
            }
            const float poison = ok ? 0.f : __int_as_float(0x7FC00000);  // a wait that ran out leaves NaN
#pragma unroll
            for (int p = 0; p < P; p++) {
                if (2 * p >= cnt)
                    break;
                const int c = 2 * p + (t >> 1);
                const long long row = (long long)sh.store_rows[min(c, cnt - 1)] * a.out_stride;
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const int n = tile * MV_TILE + g + 8 * half;
                    const float s = (half ? v[p].y : v[p].x) + bias[half] + poison;
                    const float up_raw = __shfl_down_sync(0xffffffffu, s, 4);  // row g + 1
                    if ((t & 1) == 0 && c < cnt && n < a.N) {
                        if (!a.swiglu) {
                            store_from_float(a.out, row + n, a.out_dtype, s);
                        } else if ((g & 1) == 0) {
                            const float gt = s > a.limit ? a.limit : s;  // comparisons that let NaN through
                            const float up = up_raw > a.limit ? a.limit : up_raw < -a.limit ? -a.limit : up_raw;
                            store_from_float(a.out, row + (n >> 1), a.out_dtype, gt / (1.f + expf(-a.alpha * gt)) * (up + 1.f));
                        }
                    }
                }
            }
            if (++tile == a.n_tiles) {
                tile = 0;
                li++;
            }
        }
        if (!ok)  // copies that are still on their way get a bounded time to land
            for (int i = 0; i < D; i++) {
                drain_wait(smem_u32(&sh.full[i]), 0);
                drain_wait(smem_u32(&sh.full[i]), 1);
            }
        // rows without a matrix
        if (a.ids) {
            const int n_out = a.swiglu ? a.N >> 1 : a.N;
            for (int m = 0; m < a.R; m++)
                if (sh.ids[m] < 0)
                    for (long long n = (long long)blockIdx.x * 32 + lane; n < n_out; n += (long long)gridDim.x * 32)
                        store_from_float(a.out, m * a.out_stride + n, a.out_dtype, 0.f);
        }
        return;
    }

    // ---- computes ----
    MvRun r{li0, 0, tile0, 0, 0, 0, 0};
    for (int left = i1 - i0; left > 0; r.li++, r.tile = 0) {
        // the rows of this pass, their x in fp16 and its scales
        asm volatile("bar.sync 1, %0;" ::"n"(MV_THREADS) : "memory");  // nobody computes with the last ones
        int cnt = 0;
        if (a.ids) {
            const int first = sh.rank[sh.lead[r.li]], mat = sh.ids[sh.lead[r.li]];
            for (int m0 = 0; m0 < a.R; m0 += 32) {  // every warp counts, each stores the same
                const int m = m0 + lane;
                const bool in = m < a.R && sh.ids[m] == mat && sh.rank[m] >= first && sh.rank[m] < first + RP;
                if (in)
                    sh.rows[sh.rank[m] - first] = m;
                cnt += __popc(__ballot_sync(0xffffffffu, in));
            }
        } else {
            cnt = min(RP, a.R - r.li * RP);
            if (lane < cnt)
                sh.rows[lane] = r.li * RP + lane;
        }
        __syncwarp();
        bool any = false;
        for (int c = 0; c < cnt; c++)
            any |= mv_load_x<INT4>(a, sh.rows[c] / a.rows_per_x, steps, G, reinterpret_cast<uint4*>(dyn + xs_at) + c * steps * 16,
                                   reinterpret_cast<float*>(dyn + xsc_at) + c * steps * 4);
        uint32_t far;
        asm volatile("{\n\t.reg .pred p, q;\n\t"
                     "setp.ne.u32 p, %1, 0;\n\t"
                     "bar.red.or.pred q, 1, %2, p;\n\t"
                     "selp.u32 %0, 1, 0, q;\n\t}"
                     : "=r"(far)
                     : "r"((uint32_t)any), "n"(MV_THREADS)
                     : "memory");
        const int n = min(left, a.n_tiles - r.tile);
        left -= n;
        r.cnt = cnt;
        r.tile_end = r.tile + n;
        if (__builtin_expect(far, 0)) {
            mv_tiles<INT4, PAIRED, P, true>(a, sh, dyn, r);
        } else {
            mv_tiles<INT4, PAIRED, P, false>(a, sh, dyn, r);
        }
    }
}

}  // namespace op
}  // namespace moe
