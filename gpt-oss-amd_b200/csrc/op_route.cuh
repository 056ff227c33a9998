// route_logits: expert indices and weights from router logits.
//
//   p_e = softmax_e(l) or sigmoid(l_e);  key_e = p_e + bias_e, or l_e itself without a bias (the
//   same order);  of n_groups groups only the topk_groups with the largest sum of their group_top
//   best keys take part;  the K largest keys are selected, ties to the lower index;
//   w = p of the selected (/ their sum) * scale.
//
// The indices are whole numbers and must not depend on a rounding: their order is that of keys in
// 64 bits.  Logits order exactly as they are.  Keys that are sums are computed in fp32 first, and
// a warp whose decision hung on a gap below the fp32 error does its token again with
// 64-bit keys (route_select<double>): about one token in a hundred for fp32 logits.  The weights of
// the K selected come from 64-bit exponentials, one lane each.
//
// A warp owns a token; lane i holds the NT neighbouring experts from i * NT on, so the lowest
// lane of a tie has the lowest index.  K rounds of a warp-wide maximum.  Bound by the latency of
// that chain for few tokens and by instruction issue for many; the logits are read once.
#pragma once
#include <float.h>

#include "op_types.cuh"

namespace moe {
namespace op {

constexpr int ROUTE_MAX_E = MOE_B200_ROUTE_LOGITS_MAX_EXPERTS;
constexpr int ROUTE_MAX_K = MOE_B200_ROUTE_LOGITS_MAX_K;
constexpr int ROUTE_MAX_GROUPS = 32;

struct LogitsArgs {
    const void* logits;
    long long stride;
    int dtype;
    int T, E, K;
    int sigmoid;
    const float* bias;
    int n_groups, topk_groups, group_top;
    int renorm;
    float scale;
    int* topk_i;
    float* topk_w;
    int* counts;
};

template <typename F>
__device__ __forceinline__ F warp_max(F v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const F u = __shfl_xor_sync(0xffffffffu, v, o);
        v = u > v ? u : v;
    }
    return v;
}

template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

// Largest key of the warp and the lowest expert that has it.  Keys never hold NaN.
__device__ __forceinline__ float warp_best(float v, int& e) {
    // floats as integers of the same order; -inf stays below everything
    const uint32_t b = __float_as_uint(v + 0.f);  // -0 counts as +0
    const uint32_t u = b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
    const uint32_t top = __reduce_max_sync(0xffffffffu, u);
    e = __shfl_sync(0xffffffffu, e, __ffs(__ballot_sync(0xffffffffu, u == top)) - 1);
    return __uint_as_float(top ^ ((top >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ double warp_best(double v, int& e) {
    const double top = warp_max(v);
    e = __shfl_sync(0xffffffffu, e, __ffs(__ballot_sync(0xffffffffu, v == top)) - 1);
    return top;
}

// One token.  l[j]: logit of expert lane * NT + j, -inf where it takes no part.  `keys`: E values of
// shared memory of this warp (group scores).  sel[k] in every lane; returns false where an fp32
// decision was too close to call.  sum: the softmax's (0 where nothing needs it).
template <typename F, int NT>
__device__ __forceinline__ bool route_select(const LogitsArgs& a, const float (&l)[NT], float lmax, F* keys, int lane,
                                             int* sel, F& sum) {
    // Without a bias the logits are the keys of the experts, and of groups scored by their best.
    const bool by_logit = a.bias == nullptr;
    const bool need_p = !by_logit || (a.n_groups > 1 && a.group_top > 1);
    F p[NT];
    sum = 0;
    if (!a.sigmoid && (need_p || !a.renorm)) {
#pragma unroll
        for (int j = 0; j < NT; j++) {
            p[j] = l[j] > -INFINITY ? exp_of((F)l[j] - (F)lmax) : (F)0;
            sum += p[j];
        }
        sum = warp_sum(sum);
    }
    if (need_p) {
#pragma unroll
        for (int j = 0; j < NT; j++) {
            if (a.sigmoid)
                p[j] = l[j] > -INFINITY ? (F)1 / ((F)1 + exp_of(-(F)l[j])) : (F)0;
            else
                p[j] = p[j] / sum;
        }
    }
    // Two fp32 keys closer than this may be in the other order in 64 bits: p is off by up to 48
    // half steps of its size (the exponential's two steps, the rounded difference in its argument, the
    // sum of up to 512 terms in a tree, the division), p + bias by half a step of the sum's.
    constexpr bool check = sizeof(F) == 4;
    constexpr float TOL = 2.f * 49.f * 5.97e-8f;
    bool sure = true;
    F key[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int e = lane * NT + j;
        key[j] = -INFINITY;
        if (l[j] > -INFINITY) {
            const float b = by_logit ? 0.f : a.bias[e];
            key[j] = by_logit ? (F)l[j] : b > -INFINITY ? p[j] + (F)fminf(b, FLT_MAX) : (F)-INFINITY;
        }
    }
    if (a.n_groups > 1) {
        // a group's score by the lane of its number
        const int gs = a.E / a.n_groups;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < NT; j++)
            if (lane * NT + j < a.E)
                keys[lane * NT + j] = (by_logit && a.group_top > 1 && l[j] > -INFINITY) ? p[j] : key[j];
        __syncwarp();
        F b1 = -INFINITY, b2 = -INFINITY;
        if (lane < a.n_groups)
            for (int i = 0; i < gs; i++) {
                const F v = keys[lane * gs + i];
                b2 = v > b1 ? b1 : (v > b2 ? v : b2);
                b1 = v > b1 ? v : b1;
            }
        F score = b1;
        if (a.group_top > 1 && b2 > -INFINITY)
            score += b2;
        const bool exact = by_logit && a.group_top == 1;
        unsigned kept = 0;
        F last = INFINITY;
        for (int k = 0; k <= a.topk_groups && k < a.n_groups; k++) {
            int g = lane;
            const F s = warp_best(score, g);
            if (k == a.topk_groups) {
                if (check && !exact && s > -INFINITY)
                    sure &= (float)(last - s) > 2.f * TOL * fmaxf(1.f, fabsf((float)last));
            } else if (s > -INFINITY) {
                kept |= 1u << g;
                if (lane == g)
                    score = -INFINITY;
            }
            last = s;
        }
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const int e = lane * NT + j;
            if (e < a.E && !((kept >> (e / gs)) & 1u))
                key[j] = -INFINITY;
        }
    }
    F last = INFINITY;
    for (int k = 0; k <= a.K; k++) {
        F v = key[0];
        int e = lane * NT;
#pragma unroll
        for (int j = 1; j < NT; j++)
            if (key[j] > v) {
                v = key[j];
                e = lane * NT + j;
            }
        v = warp_best(v, e);
        if (check && !by_logit && k > 0 && v > -INFINITY)
            sure &= (float)(last - v) > TOL * fmaxf(1.f, fabsf((float)last));
        last = v;
        if (k < a.K) {
            if (!(v > -INFINITY))
                e = -1;
            if (lane == 0)
                sel[k] = e;
#pragma unroll
            for (int j = 0; j < NT; j++)
                if (e == lane * NT + j)
                    key[j] = -INFINITY;
        } else if (by_logit || !check) {
            break;
        }
    }
    __syncwarp();
    return sure;
}

constexpr int ROUTE_WARPS = 4;

template <int NT>
__global__ void __launch_bounds__(32 * ROUTE_WARPS) route_logits_kernel(const LogitsArgs a) {
    __shared__ double s_keys[ROUTE_WARPS][32 * NT];
    __shared__ int s_sel[ROUTE_WARPS][ROUTE_MAX_K];
    __shared__ int s_hist[32 * NT];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (a.counts) {
        for (int i = threadIdx.x; i < a.E; i += blockDim.x)
            s_hist[i] = 0;
        __syncthreads();
    }
    for (int t = blockIdx.x * (blockDim.x >> 5) + warp; t < a.T; t += gridDim.x * (blockDim.x >> 5)) {
        float l[NT];
        float lmax = -INFINITY;
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const int e = lane * NT + j;
            l[j] = -INFINITY;
            if (e < a.E) {
                const float v = load_as_float(a.logits, (long long)t * a.stride + e, a.dtype);
                l[j] = v > -INFINITY ? fminf(v, FLT_MAX) : -INFINITY;  // NaN compares false
            }
            lmax = fmaxf(lmax, l[j]);
        }
        lmax = warp_max(lmax);
        int* sel = s_sel[warp];
        float fsum;
        double sum;
        const bool sure = route_select<float, NT>(a, l, lmax, reinterpret_cast<float*>(s_keys[warp]), lane, sel, fsum);
        sum = fsum;
        if (!sure)
            route_select<double, NT>(a, l, lmax, s_keys[warp], lane, sel, sum);
        // weights: lane k has the k-th selected
        const int e = lane < a.K ? sel[lane] : -1;
        double w = 0.0;
        if (e >= 0) {
            const float v = load_as_float(a.logits, (long long)t * a.stride + e, a.dtype);
            const double x = fminf(v, FLT_MAX);
            w = a.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - (double)lmax);
        }
        if (a.renorm)
            sum = warp_sum(w);
        if (a.renorm || !a.sigmoid)
            w = w > 0.0 ? w / sum : 0.0;
        if (lane < a.K) {
            a.topk_i[(size_t)t * a.K + lane] = e;
            a.topk_w[(size_t)t * a.K + lane] = (float)(w * (double)a.scale);
            if (a.counts && e >= 0)
                atomicAdd(&s_hist[e], 1);
        }
        __syncwarp();
    }
    if (a.counts) {
        __syncthreads();
        for (int i = threadIdx.x; i < a.E; i += blockDim.x)
            if (s_hist[i])
                atomicAdd(&a.counts[i], s_hist[i]);
    }
}

}  // namespace op
}  // namespace moe
