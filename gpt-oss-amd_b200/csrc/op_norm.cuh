// add_rmsnorm: r = x + residual, y = r * rsqrt(mean(r^2) + eps) * w, and y once more in 8 bits.
//
// Everything between the loads and the stores is fp32 and each output is rounded once; the
// norm is that of the unrounded sum.  The residual is written, the 16-bit row and the codes come
// from the same registers, so a row is read once and written once: 2 H (read) + 8 H + 2 H + H bytes
// for a bf16 x, an fp32 residual, a bf16 y and codes.  For many rows HBM bounds it (16384 x 2880 in bf16,
// fp32 residual, y, codes and row scales, 613 MB: 96 us, 6.4 TB/s), for one row the chain load -> sum over the
// block -> store (2.0 us, launch included).
//
// A block owns a row (a warp, where a warp holds it and there are many) and a thread 8 * NV columns of it in
// registers (rows of more than 16384 columns spill).  VEC: eight neighbouring columns per step, moved 16 bytes at a time (rows on 16-byte boundaries, H a
// multiple of 8).  Otherwise a warp covers the same 256 columns with eight coalesced steps of one element per lane,
// bound by issue: 777 x 2047 6.3 us, x 2048 4.1.
//
// Scales.  A group's largest |y| is found among its own lanes (a group is 4, 8 or 16 lanes with
// VEC, one, two or four steps of a warp without), a row's over the block.
#pragma once
#include "common.cuh"
#include "op_types.cuh"

namespace moe {
namespace op {

struct NormArgs {
    const void* x;
    long long x_stride;
    int x_dtype;
    const void* res;  // null: none
    void* res_out;
    long long res_stride, res_out_stride;
    int res_dtype;
    const void* w;
    int w_dtype;
    float eps;
    int n_rows, H;
    void* y;  // null: none
    long long y_stride;
    int y_dtype;
    uint8_t* q;  // null: none
    long long q_stride;
    void* scales;   // [rows, n_scales], f32 or e8m0
    int n_scales;
    int group;      // columns per scale: 32, 64, 128; 0: the row
    int group_shift;
    int mx;         // e8m0 scales
    int early;      // the next kernel's blocks may come at once
};

// Eight values of one thread, still as they were loaded.
struct Raw8 {
    uint4 a, b;
};

template <bool VEC>
__device__ __forceinline__ int norm_col(int v, int e) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int base = (v * (int)(blockDim.x >> 5) + warp) * 256;
    return VEC ? base + lane * 8 + e : base + e * 32 + lane;
}

template <bool VEC, int NV>
__device__ __forceinline__ void norm_load(Raw8 (&raw)[NV], const void* p, long long at, int dtype, int H) {
    if (VEC) {
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int c = norm_col<true>(v, 0);
            raw[v].a = raw[v].b = make_uint4(0, 0, 0, 0);
            if (c < H) {
                if (dtype == MOE_B200_DTYPE_F32) {
                    const uint4* s = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + at + c);
                    raw[v].a = s[0];
                    raw[v].b = s[1];
                } else {
                    raw[v].a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at + c);
                }
            }
        }
    } else {
#pragma unroll
        for (int v = 0; v < NV; v++) {
            uint32_t t[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int c = norm_col<false>(v, e);
                t[e] = 0;
                if (c < H)
                    t[e] = dtype == MOE_B200_DTYPE_F32 ? static_cast<const uint32_t*>(p)[at + c]
                                                       : static_cast<const uint16_t*>(p)[at + c];
            }
            raw[v].a = make_uint4(t[0], t[1], t[2], t[3]);
            raw[v].b = make_uint4(t[4], t[5], t[6], t[7]);
        }
    }
}

template <bool VEC>
__device__ __forceinline__ void norm_unpack(const Raw8& r, int dtype, float (&f)[8]) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int e = 0; e < 8; e++) {
        if (dtype == MOE_B200_DTYPE_F32)
            f[e] = __uint_as_float(w[e]);
        else if (VEC)
            f[e] = half_to_float((w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu, dtype);
        else
            f[e] = half_to_float(w[e], dtype);
    }
}

template <bool VEC>
__device__ __forceinline__ void norm_store(void* p, long long at, int dtype, int H, int v, const float (&f)[8]) {
    if (VEC) {
        const int c = norm_col<true>(v, 0);
        if (c >= H)
            return;
        if (dtype == MOE_B200_DTYPE_F32) {
            float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + at + c);
            d[0] = make_float4(f[0], f[1], f[2], f[3]);
            d[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + at + c) =
                make_uint4(floats_to_half2(f[0], f[1], dtype), floats_to_half2(f[2], f[3], dtype),
                           floats_to_half2(f[4], f[5], dtype), floats_to_half2(f[6], f[7], dtype));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int c = norm_col<false>(v, e);
            if (c < H)
                store_from_float(p, at + c, dtype, f[e]);
        }
    }
}

// Sum / maximum over the block, the same value in every thread.  `slots`: 32 floats of shared
// memory that no other call uses.  Lanes and warps are added in a fixed order.
template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float* slots) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float u = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? fmaxf(v, u) : v + u;
    }
    const int warps = blockDim.x >> 5;
    if (warps == 1)
        return v;
    if ((threadIdx.x & 31) == 0)
        slots[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (int)(threadIdx.x & 31) < warps ? slots[threadIdx.x & 31] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float u = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? fmaxf(v, u) : v + u;
    }
    return v;
}

// Exponent byte of the least power of two s with amax <= 448 s, 448 = 1.75 * 2^8: read off the
// bits of amax, so a value on the border decides exactly.  0 gives 2^0.
__device__ __forceinline__ uint32_t mx_scale_byte(float amax) {
    const uint32_t b = __float_as_uint(amax);
    if (b == 0)
        return 127;
    const int e = (int)(b >> 23) - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return (uint32_t)min(max(e, 0), 254);
}

// 1 / scale and the scale itself, as stored, from a group's largest |y|.  A code is that of y * (1 / scale): one rounding
// of fp32 more than y / scale, which puts one code in 1.7 million on the neighbouring value (MX: none, the reciprocal is
// exact).  Two more operations per element that take it back cost 1.3 % of 16384 x 2880, 6.5 % of 777 x 2047.
__device__ __forceinline__ float norm_put_scale(const NormArgs& a, long long i, float amax, bool store) {
    if (a.mx) {
        const uint32_t byte = mx_scale_byte(amax);
        if (store)
            static_cast<uint8_t*>(a.scales)[i] = (uint8_t)byte;
        return __uint_as_float(max((254u - byte) << 23, 0x00400000u));  // 2^(127 - byte)
    }
    const float s = amax > 0.f ? fmaxf(amax / 448.f, 1.17549435e-38f) : 1.f;  // its reciprocal is finite
    if (store)
        static_cast<float*>(a.scales)[i] = s;
    return 1.f / s;
}

template <bool VEC, int NV>
__global__ void __launch_bounds__(1024) add_rmsnorm_kernel(const NormArgs a) {
    __shared__ float slots[64];
    pdl_wait();
    if (a.early)
        pdl_trigger();
    const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;  // blockDim.y > 1: a warp per row
    if (row >= a.n_rows)
        return;
    const int H = a.H;
    const int lane = threadIdx.x & 31;
    float r[NV][8];
    Raw8 wr[NV];
    {
        Raw8 xr[NV], rr[NV];
        norm_load<VEC, NV>(xr, a.x, row * a.x_stride, a.x_dtype, H);
        if (a.res)
            norm_load<VEC, NV>(rr, a.res, row * a.res_stride, a.res_dtype, H);
        norm_load<VEC, NV>(wr, a.w, 0, a.w_dtype, H);
#pragma unroll
        for (int v = 0; v < NV; v++) {
            norm_unpack<VEC>(xr[v], a.x_dtype, r[v]);
            if (a.res) {
                float t[8];
                norm_unpack<VEC>(rr[v], a.res_dtype, t);
#pragma unroll
                for (int e = 0; e < 8; e++)
                    r[v][e] += t[e];
                if (a.res_out)
                    norm_store<VEC>(a.res_out, row * a.res_out_stride, a.res_dtype, H, v, r[v]);
            }
        }
    }
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < NV; v++)
#pragma unroll
        for (int e = 0; e < 8; e++)
            ss = fmaf(r[v][e], r[v][e], ss);  // columns past H hold zeros
    ss = block_reduce<false>(ss, slots);
    const float rinv = 1.f / sqrtf(ss / (float)H + a.eps);
    float top = 0.f;
#pragma unroll
    for (int v = 0; v < NV; v++) {
        float t[8];
        norm_unpack<VEC>(wr[v], a.w_dtype, t);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            r[v][e] = r[v][e] * rinv * t[e];
            top = fmaxf(top, fabsf(r[v][e]));
        }
        if (a.y)
            norm_store<VEC>(a.y, row * a.y_stride, a.y_dtype, H, v, r[v]);
    }
    if (!a.q)
        return;
    float inv_row = 0.f;
    if (a.group == 0) {
        top = block_reduce<true>(top, slots + 32);
        inv_row = norm_put_scale(a, row, top, threadIdx.x == 0);
    }
    uint8_t* q = a.q + row * a.q_stride;
    const long long s0 = row * a.n_scales;
#pragma unroll
    for (int v = 0; v < NV; v++) {
        if (VEC) {
            float inv = inv_row;
            const int c = norm_col<true>(v, 0);
            if (a.group) {
                float m = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++)
                    m = fmaxf(m, fabsf(r[v][e]));
                for (int o = 1; o < a.group / 8; o <<= 1)
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                inv = norm_put_scale(a, s0 + (c >> a.group_shift), m, c < H && (c & (a.group - 1)) == 0);
            }
            if (c < H) {
                uint2 d;
                d.x = floats_to_e4m3x2(r[v][0] * inv, r[v][1] * inv) | floats_to_e4m3x2(r[v][2] * inv, r[v][3] * inv) << 16;
                d.y = floats_to_e4m3x2(r[v][4] * inv, r[v][5] * inv) | floats_to_e4m3x2(r[v][6] * inv, r[v][7] * inv) << 16;
                *reinterpret_cast<uint2*>(q + c) = d;
            }
        } else {
            // a group is one, two or four steps of a warp
            float inv[8];
#pragma unroll
            for (int e = 0; e < 8; e++)
                inv[e] = inv_row;
            if (a.group) {
                float m[8];
#pragma unroll
                for (int e = 0; e < 8; e++)  // non-negative floats order like their bits; NaN counts as 0
                    m[e] = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fabsf(r[v][e]), 0.f))));
                const int c0 = norm_col<false>(v, 0) - lane;
                auto scale_of = [&](int e, float top) {
                    const int c = c0 + e * 32;
                    return norm_put_scale(a, s0 + (c >> a.group_shift), top, lane == 0 && c < H);
                };
                if (a.group == 32) {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        inv[e] = scale_of(e, m[e]);
                } else if (a.group == 64) {
#pragma unroll
                    for (int e = 0; e < 8; e += 2)
                        inv[e] = inv[e + 1] = scale_of(e, fmaxf(m[e], m[e + 1]));
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e += 4)
                        inv[e] = inv[e + 1] = inv[e + 2] = inv[e + 3] =
                            scale_of(e, fmaxf(fmaxf(m[e], m[e + 1]), fmaxf(m[e + 2], m[e + 3])));
                }
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int c = norm_col<false>(v, e);
                if (c < H)
                    q[c] = (uint8_t)(floats_to_e4m3x2(r[v][e] * inv[e], 0.f) & 0xFFu);
            }
        }
    }
}

}  // namespace op
}  // namespace moe
