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
// Ring stages of a warp (two steps of 128 columns each) and blocks per SM with P pairs of x rows: as much in
// flight as shared memory and registers hold.
__host__ __device__ constexpr int mv_depth(int P) { return P == 4 ? 2 : 3; }
constexpr int MV_BLOCKS = 2;
constexpr int MV_STAGE_BYTES = 2 * 1024 + 256;                // per step: codes of rows 0..7, of rows 8..15; scale words
constexpr int MV_DIRECT = 3;                                  // SH: scales are loaded where they are used
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
    int ksplit;             // warps that share a tile: 1, 2, 4 or 8, at most the stages of a row
};

// Dynamic shared memory: zeros, the rings of the warps, x rows in fp16, then their scales per group of 32.
__host__ __device__ constexpr int mv_x_at(int P) { return 64 + MV_WARPS * mv_depth(P) * MV_STAGE_BYTES; }
__host__ __device__ constexpr int mv_steps(int K) { return (K + 127) / 128; }
__host__ __device__ constexpr size_t mv_smem_bytes(int K, int P, int rows) {
    return mv_x_at(P) + (size_t)rows * mv_steps(K) * (128 * 2 + 4 * 4);
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
// 1 of the result, int4: its halves.
template <bool INT4>
__device__ __forceinline__ uint32_t mv_load_scales(const uint8_t* row, int sg, int G, int shift) {
    uint32_t r = 0;
    if (INT4) {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
        if (sg < G)
            r = p[sg >> shift];
        if (sg + 1 < G)
            r |= (uint32_t)p[(sg + 1) >> shift] << 16;
    } else {
        if (sg < G)
            r = row[sg];
        if (sg + 1 < G)
            r |= (uint32_t)row[sg + 1] << 8;
    }
    return r;
}

// The same from the words of a stage.  A stage's scales start at byte `o` of a row's four words; mv_pick is
// the byte selector of a lane for its first step, mv_from_words applies it for step h.
template <bool INT4, int SH>
__device__ __forceinline__ uint32_t mv_pick(const uint8_t* at, int t) {
    const uint32_t o = (uint32_t)(reinterpret_cast<uintptr_t>(at) & 3), k = t & 1;
    if (!INT4)
        return (o + 2 * k) * 0x11u + 0x7710u;  // bytes 2 and 3 of the result are not used
    if (SH == 0)
        return k ? 0x7654u : 0x3210u;
    return (SH == 1 ? o + 2 * k : o) * 0x1111u + 0x1010u;
}
template <bool INT4, int SH>
__device__ __forceinline__ uint32_t mv_from_words(const uint4& w, uint32_t pick, int h) {
    if (INT4 && SH == 0)
        return h ? __byte_perm(w.z, w.w, pick) : __byte_perm(w.x, w.y, pick);
    if (INT4 && SH == 2)
        return __byte_perm(w.x, w.y, pick + 0x2222u * h);
    return h ? __byte_perm(w.y, w.z, pick) : __byte_perm(w.x, w.y, pick);
}

__device__ __forceinline__ void mv_copy16(int at, const void* src) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(at), "l"(src) : "memory");
}
__device__ __forceinline__ void mv_copy4(int at, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at), "l"(src) : "memory");
}
__device__ __forceinline__ void mv_copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void mv_copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// P pairs of x rows (columns of the MMA) per pass over the weights.
// SH: log2 of 32-column groups per scale, the scales coming through the ring in aligned words; MV_DIRECT where they
// cannot (an odd number of bf16 scales per row, or scales off a word boundary).
template <bool INT4, int SH, int P>
__global__ void __launch_bounds__(MV_THREADS, MV_BLOCKS) w4_matvec_kernel(const MatvecArgs a) {
    constexpr int RP = 2 * P, DEPTH = mv_depth(P);
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ int s_ids[MV_MAX_ROWS];
    __shared__ int s_lead[MV_MAX_ROWS];
    __shared__ int s_rank[MV_MAX_ROWS];
    __shared__ int s_warp_cnt[MV_WARPS];
    __shared__ int s_rows[RP];
    __shared__ float2 s_red[2][MV_WARPS][P][16];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int steps = mv_steps(a.K), G = a.K >> 5, SG = G >> a.group_shift;
    const int xs_at = mv_x_at(P), xsc_at = xs_at + min(RP, a.R) * steps * 256;
    uint4* xs = reinterpret_cast<uint4*>(dyn + xs_at);
    float* xsc = reinterpret_cast<float*>(dyn + xsc_at);
    if (tid < 4)
        reinterpret_cast<uint4*>(dyn)[tid] = make_uint4(0, 0, 0, 0);

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
    const int KS = a.ksplit, ks = warp & (KS - 1), slot = warp / KS, n_slots = MV_WARPS / KS;
    const int half = (steps + 1) >> 1;  // stages of a row
    const int b0 = 2 * (half * ks / KS), b1 = min(2 * (half * (ks + 1) / KS), steps);  // never empty
    constexpr int SB = INT4 ? 2 : 1;  // bytes of a scale
    const int ring_off = 64 + warp * DEPTH * MV_STAGE_BYTES + lane * 16;
    const int ring_at = (int)__cvta_generic_to_shared(dyn) + ring_off, at_words = ring_at - lane * 12 + 2048;
    const uint8_t* s_last = static_cast<const uint8_t*>(a.scales) + (size_t)a.n_mats * a.N * SG * SB - 4;  // last whole word
    const bool quad_b = (g & 3) == t;  // lanes of the block diagonal of B

    int buf = 0;
    for (int item = i0; item < i1;) {
        // a run of tiles of one matrix for the same rows of x
        const int li = item / a.n_tiles, ta = item % a.n_tiles, tb = min(a.n_tiles, ta + i1 - item);
        item += tb - ta;
        const int mat = a.ids ? s_ids[s_lead[li]] : 0;
        const uint8_t* codes = a.codes + (size_t)mat * a.N * G * 16;
        const uint8_t* scales = static_cast<const uint8_t*>(a.scales) + (size_t)mat * a.N * SG * SB;
        const int n_mine = ta + slot < tb ? (tb - ta - slot + n_slots - 1) / n_slots : 0;




        // The codes run DEPTH - 1 stages ahead, into the next tile too.  Rows past the end read the last row (and
        // are not stored); groups past the end are not loaded: what the stage held is finite, and their x is zero.
        const int g_end = min(G, b1 * 4);
        int l_left = n_mine * ((b1 - b0 + 1) >> 1), l_tile = ta + slot, l_g = b0 * 4 + t, l_stage = 0;
        const uint8_t *c_lo, *c_hi, *w_lo_at, *w_hi_at;
        auto start_tile = [&]() {
            const int r_lo = min(l_tile * MV_TILE + g, a.N - 1), r_hi = min(l_tile * MV_TILE + g + 8, a.N - 1);
            c_lo = codes + (size_t)r_lo * G * 16 + (b0 * 4 + t) * 16;
            c_hi = codes + (size_t)r_hi * G * 16 + (b0 * 4 + t) * 16;
            l_g = b0 * 4 + t;
            if (SH != MV_DIRECT) {  // lane t copies word t
                w_lo_at = scales + ((size_t)r_lo * SG + ((b0 * 4) >> SH)) * SB;
                w_hi_at = scales + ((size_t)r_hi * SG + ((b0 * 4) >> SH)) * SB;
                w_lo_at += 4 * t - (reinterpret_cast<uintptr_t>(w_lo_at) & 3);
                w_hi_at += 4 * t - (reinterpret_cast<uintptr_t>(w_hi_at) & 3);
            }
        };
        auto load = [&]() {
            if (l_left > 0) {
                const int at = ring_at + l_stage;
                if (l_g < g_end) {
                    mv_copy16(at, c_lo);
                    mv_copy16(at + 512, c_hi);
                }
                if (l_g + 4 < g_end) {
                    mv_copy16(at + 1024, c_lo + 64);
                    mv_copy16(at + 1536, c_hi + 64);
                }
                if (SH != MV_DIRECT) {
                    // what these words hold behind the scales of the stage is not used
                    const bool mine = t < (INT4 ? (SH == 0 ? 4 : SH == 1 ? 3 : 2) : 3);
                    if (mine && w_lo_at <= s_last)
                        mv_copy4(at_words + l_stage, w_lo_at);
                    if (mine && w_hi_at <= s_last)
                        mv_copy4(at_words + l_stage + 128, w_hi_at);
                    w_lo_at += (8 * SB) >> SH;
                    w_hi_at += (8 * SB) >> SH;
                }
                c_lo += 128;
                c_hi += 128;
                l_g += 8;
                l_left--;
                if (l_g - t >= b1 * 4) {
                    l_tile += n_slots;
                    start_tile();
                }
            }
            l_stage = l_stage == (DEPTH - 1) * MV_STAGE_BYTES ? 0 : l_stage + MV_STAGE_BYTES;
            mv_copies_commit();
        };
        start_tile();
#pragma unroll 1
        for (int i = 0; i < DEPTH - 1; i++)
            load();

        // the rows of this pass, their x in fp16 and its scales
        int cnt;
        __syncthreads();  // the previous run has been computed
        if (a.ids) {
            const int first = s_rank[s_lead[li]];
            const bool in = tid < a.R && s_ids[tid] == mat && s_rank[tid] >= first && s_rank[tid] < first + RP;
            if (in)
                s_rows[s_rank[tid] - first] = tid;
            cnt = __syncthreads_count(in);
        } else {
            cnt = min(RP, a.R - li * RP);
            if (tid < cnt)
                s_rows[tid] = li * RP + tid;
            __syncthreads();
        }
        for (int c = 0; c < cnt; c++) {
            const long long xr = s_rows[c] / a.rows_per_x;
            for (int k8 = tid; k8 < steps * 16; k8 += MV_THREADS) {  // eight columns; four lanes make a group
                const int grp = k8 >> 2;
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
                xs[c * steps * 16 + k8] = make_uint4(h[0], h[1], h[2], h[3]);
                if ((k8 & 3) == 0)
                    xsc[c * steps * 4 + grp] = sc;
            }
        }
        __syncthreads();

        float acc[P][4];
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int k = 0; k < 4; k++)
                acc[p][k] = 0.f;
        // Lanes off the diagonal, and those of x rows that are not there, read zeros.
        int x_at[P], x_step[P], sc_at[P];
#pragma unroll
        for (int p = 0; p < P; p++) {
            const int c = 2 * p + (g >> 2), cs = 2 * p + (t >> 1);
            const bool mine = quad_b && c < cnt;
            x_at[p] = mine ? xs_at + (c * steps * 16 + t * 4) * 16 : 0;
            x_step[p] = mine ? 256 : 0;
            sc_at[p] = xsc_at + (min(cs, cnt - 1) * steps * 4 + 2 * (t & 1)) * 4;
        }
        int stage = 0;
        for (int tile = ta + slot; tile < tb; tile += n_slots) {
            const uint8_t* s_lo = scales + (size_t)min(tile * MV_TILE + g, a.N - 1) * SG * SB;
            const uint8_t* s_hi = scales + (size_t)min(tile * MV_TILE + g + 8, a.N - 1) * SG * SB;
            uint32_t pick_lo = 0, pick_hi = 0;
            if (SH != MV_DIRECT) {
                pick_lo = mv_pick<INT4, SH>(s_lo + ((b0 * 4) >> SH) * SB, t);
                pick_hi = mv_pick<INT4, SH>(s_hi + ((b0 * 4) >> SH) * SB, t);
            }
#pragma unroll 1
            for (int b = b0; b < b1; b += 2) {
                mv_copies_wait<DEPTH - 2>();
                __syncwarp();  // every lane's copies have landed, and the stage before this one has been read
                load();
                const uint8_t* st = dyn + ring_off + stage;
                uint4 words_lo, words_hi;
                if (SH != MV_DIRECT) {
                    const uint8_t* sw = dyn + ring_off - lane * 16 + 2048 + g * 16 + stage;
                    words_lo = *reinterpret_cast<const uint4*>(sw);
                    words_hi = *reinterpret_cast<const uint4*>(sw + 128);
                }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint4 c_lo4 = *reinterpret_cast<const uint4*>(st + h * 1024);
                    const uint4 c_hi4 = *reinterpret_cast<const uint4*>(st + h * 1024 + 512);
                    const uint32_t w_lo[4] = {c_lo4.x, c_lo4.y, c_lo4.z, c_lo4.w};
                    const uint32_t w_hi[4] = {c_hi4.x, c_hi4.y, c_hi4.z, c_hi4.w};
                    uint32_t l[4][4], u[4][4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        mv_decode<INT4>(w_lo[k], l[k]);
                        mv_decode<INT4>(w_hi[k], u[k]);
                    }
                    uint32_t raw_lo, raw_hi;
                    if (SH != MV_DIRECT) {
                        raw_lo = mv_from_words<INT4, SH>(words_lo, pick_lo, h);
                        raw_hi = mv_from_words<INT4, SH>(words_hi, pick_hi, h);
                        if ((b + h) * 4 + 4 > g_end) {  // what lies behind the last scale is not this row's, and may be NaN
                            const int left = g_end - (b + h) * 4 - 2 * (t & 1);
                            const uint32_t own = left > 1 ? 0xFFFFFFFFu : left == 1 ? (INT4 ? 0xFFFFu : 0xFFu) : 0u;
                            raw_lo &= own;
                            raw_hi &= own;
                        }
                    } else {
                        raw_lo = mv_load_scales<INT4>(s_lo, (b + h) * 4 + 2 * (t & 1), g_end, a.group_shift);
                        raw_hi = mv_load_scales<INT4>(s_hi, (b + h) * 4 + 2 * (t & 1), g_end, a.group_shift);
                    }
                    const float2 w_s_lo = mv_scales<INT4>(raw_lo), w_s_hi = mv_scales<INT4>(raw_hi);
                    // The second step of the last stage may not be this warp's: its x counts as zero.
                    const bool there = h == 0 || b + 1 < b1;
#pragma unroll
                    for (int p = 0; p < P; p++) {
                        if (P > 1 && 2 * p >= cnt)
                            break;
                        const uint4* x = reinterpret_cast<const uint4*>(dyn + (there ? x_at[p] + x_step[p] * (b + h) : 0));
                        const uint4 x0 = x[0], x1 = x[1], x2 = x[2], x3 = x[3];
                        float d[4];
                        mv_mma_first(d, l[0][0], u[0][0], l[0][1], u[0][1], x0.x, x0.y);
                        mv_mma(d, l[0][2], u[0][2], l[0][3], u[0][3], x0.z, x0.w);
                        mv_mma(d, l[1][0], u[1][0], l[1][1], u[1][1], x1.x, x1.y);
                        mv_mma(d, l[1][2], u[1][2], l[1][3], u[1][3], x1.z, x1.w);
                        mv_mma(d, l[2][0], u[2][0], l[2][1], u[2][1], x2.x, x2.y);
                        mv_mma(d, l[2][2], u[2][2], l[2][3], u[2][3], x2.z, x2.w);
                        mv_mma(d, l[3][0], u[3][0], l[3][1], u[3][1], x3.x, x3.y);
                        mv_mma(d, l[3][2], u[3][2], l[3][3], u[3][3], x3.z, x3.w);
                        // the product with the x scale first: the two scales alone may leave fp32
                        const float2 sx = *reinterpret_cast<const float2*>(dyn + (there ? sc_at[p] + 16 * (b + h) : 0));
                        acc[p][0] = fmaf(d[0] * sx.x, w_s_lo.x, acc[p][0]);
                        acc[p][1] = fmaf(d[1] * sx.y, w_s_lo.y, acc[p][1]);
                        acc[p][2] = fmaf(d[2] * sx.x, w_s_hi.x, acc[p][2]);
                        acc[p][3] = fmaf(d[3] * sx.y, w_s_hi.y, acc[p][3]);
                    }
                }
                stage = stage == (DEPTH - 1) * MV_STAGE_BYTES ? 0 : stage + MV_STAGE_BYTES;
            }

            // the end of a tile: rows g and g + 8 of x row 2 p + t / 2, two groups here, two with lane t ^ 1
            float lo[P], hi[P];
#pragma unroll
            for (int p = 0; p < P; p++) {
                lo[p] = acc[p][0] + acc[p][1];
                hi[p] = acc[p][2] + acc[p][3];
                lo[p] += __shfl_xor_sync(0xffffffffu, lo[p], 1);
                hi[p] += __shfl_xor_sync(0xffffffffu, hi[p], 1);
                acc[p][0] = acc[p][1] = acc[p][2] = acc[p][3] = 0.f;
            }
            if (KS > 1) {
                if (ks > 0 && (t & 1) == 0)
#pragma unroll
                    for (int p = 0; p < P; p++)
                        s_red[buf][warp][p][lane >> 1] = make_float2(lo[p], hi[p]);
                asm volatile("bar.sync %0, %1;" ::"r"(1 + slot), "r"(32 * KS) : "memory");
                if (ks == 0)
                    for (int w = 1; w < KS; w++)
#pragma unroll
                        for (int p = 0; p < P; p++) {
                            const float2 v = s_red[buf][warp + w][p][lane >> 1];
                            lo[p] += v.x;
                            hi[p] += v.y;
                        }
                buf ^= 1;
            }
            if (ks == 0) {
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const int n = tile * MV_TILE + g + 8 * half;
                    const float bias = a.bias && n < a.N ? a.bias[(size_t)mat * a.N + n] : 0.f;
#pragma unroll
                    for (int p = 0; p < P; p++) {
                        const float v = (half ? hi[p] : lo[p]) + bias;
                        const float up = __shfl_down_sync(0xffffffffu, v, 4);  // row g + 1
                        const int c = 2 * p + (t >> 1);
                        if ((t & 1) == 0 && c < cnt && n < a.N) {
                            const long long row = (long long)s_rows[c] * a.out_stride;
                            if (!a.swiglu) {
                                store_from_float(a.out, row + n, a.out_dtype, v);
                            } else if ((g & 1) == 0) {
                                const float gt = v > a.limit ? a.limit : v;  // comparisons that let NaN through
                                const float u = up > a.limit ? a.limit : up < -a.limit ? -a.limit : up;
                                store_from_float(a.out, row + (n >> 1), a.out_dtype, gt / (1.f + expf(-a.alpha * gt)) * (u + 1.f));
                            }
                        }
                    }
                }
            }
        }
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
