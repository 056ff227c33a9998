// route_logits: expert indices and weights from router logits.
//
//   p_e = softmax_e(l) or sigmoid(l_e);  key_e = p_e + bias_e, or l_e itself without a bias (the
//   same order);  of n_groups groups only the topk_groups with the largest sum of their group_top
//   best keys take part;  the K largest keys are selected, ties to the lower index;
//   w = p of the selected (/ their sum) * scale.
//
// The indices are whole numbers and must not depend on a rounding: their order is that of keys in
// 64 bits.  Logits order exactly as they are.  Keys that are sums are computed in fp32 first, and
// a warp whose decision hung on a gap below the fp32 error ranks those that may be among the K by
// 64-bit keys, a few tokens in a thousand for fp32 logits; where it hung on the groups, or on more
// than 32 experts, it does the token again in 64 bits (route_exact).
//
// A warp owns a token; a lane holds NT neighbouring experts, lanes and experts in the same order, so the lowest
// lane of a tie has the lowest index.  Where NT allows it every group has 2^n lanes of its own, the last of them
// empty if need be, and is scored and dropped by lanes (240 experts in 4 groups, 4096 tokens: 11.6 us without,
// 7.8 with).  Each lane puts its keys in order once, by counting for each the keys in front of it; then a round
// per selected expert takes the largest of the 32 heads (one warp reduction) and the winner moves on to its next
// key.  The logits are read once, 16 bytes a lane where they are aligned.
//
// Bound by instruction issue for many tokens: 749 instructions per token of 256 experts with bias, top 8,
// 16384 tokens in 16.0 us with fp32 logits (16.8 MB, 2.5 us at the HBM rate).  The order by a sorting
// network of 19 exchanges took 19.1, a search over all keys per round 44.  Few tokens are bound by
// the latency of load, order and rounds: one token 2.2 us, launch included.
#pragma once
#include <float.h>

#include "common.cuh"
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
    int lane_shift, lane_groups, lane_size;  // 2^lane_shift lanes for each of lane_groups groups of lane_size experts
    int renorm;
    float scale;
    int* topk_i;
    float* topk_w;
    int* counts;
    int early;  // the next kernel's blocks may come at once
};

__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const double u = __shfl_xor_sync(0xffffffffu, v, o);
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

// Largest value of the warp.  Keys never hold NaN.
__device__ __forceinline__ float warp_best(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// The logit that takes part: NaN and -inf do not (-inf), +inf is the largest finite value.
__device__ __forceinline__ float route_logit(float v) { return fminf(fmaxf(v, -INFINITY), FLT_MAX); }

// One token with 64-bit keys, from the definition and without hurry: `keys` holds E values of shared memory of
// this warp.  Returns the expert of slot `lane`, -1 where there is none.
__device__ __noinline__ int route_exact(const LogitsArgs& a, long long t, float lmax, double* keys, int lane) {
    const long long at = t * a.stride;
    double sum = 0.0;
    if (!a.sigmoid)
        for (int e = lane; e < a.E; e += 32) {
            const float l = route_logit(load_as_float(a.logits, at + e, a.dtype));
            if (l > -INFINITY)
                sum += exp((double)l - (double)lmax);
        }
    sum = warp_sum(sum);
    for (int e = lane; e < a.E; e += 32) {
        const float l = route_logit(load_as_float(a.logits, at + e, a.dtype));
        const float b = a.bias ? a.bias[e] : 0.f;
        double p = -INFINITY;
        if (l > -INFINITY && b > -INFINITY) {
            p = a.sigmoid ? 1.0 / (1.0 + exp(-(double)l)) : exp((double)l - (double)lmax) / sum;
            p += (double)fminf(b, FLT_MAX);
        }
        keys[e] = p;  // without a bias p itself: the groups' scores
    }
    __syncwarp();
    unsigned kept = 0xffffffffu;
    const int gs = a.E / a.n_groups;
    if (a.n_groups > 1) {
        double b1 = -INFINITY, b2 = -INFINITY;
        if (lane < a.n_groups)
            for (int i = 0; i < gs; i++) {
                const double v = keys[lane * gs + i];
                b2 = v > b1 ? b1 : (v > b2 ? v : b2);
                b1 = v > b1 ? v : b1;
            }
        double score = a.group_top > 1 && b2 > -INFINITY ? b1 + b2 : b1;
        kept = 0;
        for (int k = 0; k < a.topk_groups; k++) {
            const double top = warp_max(score);
            const int g = __ffs(__ballot_sync(0xffffffffu, score == top)) - 1;
            if (top > -INFINITY)
                kept |= 1u << g;
            if (lane == g)
                score = -INFINITY;
        }
    }
    for (int e = lane; e < a.E; e += 32) {
        if (!((kept >> (e / gs)) & 1u))
            keys[e] = -INFINITY;
        else if (!a.bias)  // the logits order the experts
            keys[e] = route_logit(load_as_float(a.logits, at + e, a.dtype));
    }
    __syncwarp();
    int mine = -1;
    for (int k = 0; k < a.K; k++) {
        double v = -INFINITY;
        int e = a.E;
        for (int i = lane; i < a.E; i += 32)
            if (keys[i] > v) {
                v = keys[i];
                e = i;
            }
        const double top = warp_max(v);
        const int win = (int)__reduce_min_sync(0xffffffffu, v == top ? (unsigned)e : 0xffffffffu);
        if (!(top > -INFINITY))
            break;
        if (lane == k)
            mine = win;
        if (lane == (win & 31))
            keys[win] = -INFINITY;
        __syncwarp();
    }
    return mine;
}

// In fp32, 0 for -inf: relative error 2^-21 + |x| 2^-23 at most.
__device__ __forceinline__ float route_sigmoid(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + __expf(-x)));
    return r;
}

// Tokens of a block.  Microseconds of 256 experts, bias, top 8 with blocks of 1, 4 and 16 warps: 64 tokens 4.1, 4.1,
// 5.0; 2048 5.6, 5.4, 5.5; 4736 9.2, 7.8, 7.6; 16384 20.7, 17.0, 17.6.  Registers for eight blocks of 4 per SM: 16.0.
constexpr int ROUTE_WARPS = 4;

// Places of N of a lane's keys in falling order, ties by index, four bits each: a key's place is the number of keys
// in front of it, and a comparison of two moves one of them a place back.
template <int N>
__device__ __forceinline__ void places_of(const float* key, int* place) {
    unsigned packed = 0;
#pragma unroll
    for (int i = 0; i < N; i++)
        packed |= (unsigned)(N - 1 - i) << (4 * i);
#pragma unroll
    for (int j = 1; j < N; j++)
#pragma unroll
        for (int i = 0; i < j; i++)
            if (key[i] >= key[j])
                packed += (1u << (4 * j)) - (1u << (4 * i));
#pragma unroll
    for (int i = 0; i < N; i++)
        place[i] = (int)(packed >> (4 * i)) & 15;
}

// A lane's keys lie in lists of up to 8 in order: 16 keys in one list are 120 comparisons, in two 56 and a comparison
// of their heads per round (4096 tokens, 304 experts, top 10: 11.1 us, 9.4).
template <int NT>
struct RouteLists {
    static constexpr int N = NT < 8 ? NT : 8, LISTS = NT / N, ROWS = LISTS * (N + 1);  // each with -inf at its end
};

// Dynamic shared memory of a warp: its keys in order, and route_exact's.
template <int NT>
__host__ __device__ constexpr size_t route_smem_bytes() {
    return RouteLists<NT>::ROWS * 32 * sizeof(float2) + NT * 32 * sizeof(double);
}

// VEC: a lane's logits are one aligned piece of memory.  (NT = 16 with its 96 registers keeps 52 bytes in local memory.)
template <int NT, bool VEC>
__global__ void __launch_bounds__(32 * ROUTE_WARPS, NT == 16 ? 5 : 8) route_logits_kernel(const __grid_constant__ LogitsArgs a) {
    __shared__ int s_sel[ROUTE_WARPS][32];
    extern __shared__ double s_dyn[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float2(*sorted)[32] = reinterpret_cast<float2(*)[32]>(s_dyn + warp * (route_smem_bytes<NT>() / 8));  // place, lane
    double* s_keys = reinterpret_cast<double*>(sorted + RouteLists<NT>::ROWS);
    pdl_wait();
    if (a.early)
        pdl_trigger();
    if (a.counts && blockIdx.x == 0)
        for (int i = threadIdx.x; i < a.E; i += 32 * ROUTE_WARPS)
            a.counts[i] = 0;  // route_counts_kernel adds to them
    // Without a bias the logits are the keys of the experts, and of groups that are scored by their best.
    const bool by_logit = a.bias == nullptr;
    const bool need_p = !by_logit || (a.n_groups > 1 && a.group_top > 1);
    const int gs = a.E / a.n_groups, span = 1 << a.lane_shift;
    const bool lanes_of_group = a.lane_groups == a.n_groups;
    // this lane's experts: `have` from e0 on
    const int in_group = (lane & (span - 1)) * NT, e0 = (lane >> a.lane_shift) * a.lane_size + in_group;
    const int have = lane >> a.lane_shift < a.lane_groups ? min(max(a.lane_size - in_group, 0), NT) : 0;
    float bias[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const float b = a.bias && j < have ? a.bias[e0 + j] : 0.f;
        bias[j] = b > -INFINITY ? fminf(b, FLT_MAX) : -INFINITY;
    }
    constexpr int LN = RouteLists<NT>::N, LISTS = RouteLists<NT>::LISTS;
#pragma unroll
    for (int i = 0; i < LISTS; i++)
        sorted[i * (LN + 1) + LN][lane] = make_float2(-INFINITY, 0.f);
    int* sel = s_sel[warp];
    for (int t = blockIdx.x * ROUTE_WARPS + warp; t < a.T; t += gridDim.x * ROUTE_WARPS) {
        float l[NT];
        const long long at = (long long)t * a.stride;
        if (VEC && have == NT) {
            if (a.dtype == MOE_B200_DTYPE_F32) {
                const float* src = static_cast<const float*>(a.logits) + at + e0;
                if (NT >= 4) {
#pragma unroll
                    for (int j = 0; j < NT; j += 4) {
                        const float4 v = *reinterpret_cast<const float4*>(src + j);
                        l[j] = v.x, l[(j + 1) % NT] = v.y, l[(j + 2) % NT] = v.z, l[(j + 3) % NT] = v.w;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < NT; j++)
                        l[j] = src[j];
                }
            } else {
                const uint16_t* src = static_cast<const uint16_t*>(a.logits) + at + e0;
                uint32_t w[(NT + 1) / 2];
                if (NT >= 8) {
#pragma unroll
                    for (int j = 0; j < NT / 2; j += 4) {
                        const uint4 v = *reinterpret_cast<const uint4*>(src + 2 * j);
                        w[j] = v.x, w[(j + 1) % ((NT + 1) / 2)] = v.y, w[(j + 2) % ((NT + 1) / 2)] = v.z, w[(j + 3) % ((NT + 1) / 2)] = v.w;
                    }
                } else if (NT == 4) {
                    const uint2 v = *reinterpret_cast<const uint2*>(src);
                    w[0] = v.x, w[1 % ((NT + 1) / 2)] = v.y;
                } else if (NT == 2) {
                    w[0] = *reinterpret_cast<const uint32_t*>(src);
                } else {
                    w[0] = *src;
                }
#pragma unroll
                for (int j = 0; j < NT; j++)
                    l[j] = half_to_float((w[j >> 1] >> (16 * (j & 1))) & 0xFFFFu, a.dtype);
            }
        } else {
#pragma unroll
            for (int j = 0; j < NT; j++)
                l[j] = j < have ? load_as_float(a.logits, at + e0 + j, a.dtype) : -INFINITY;
        }
        float lmax = -INFINITY;
#pragma unroll
        for (int j = 0; j < NT; j++) {
            l[j] = route_logit(l[j]);
            lmax = fmaxf(lmax, l[j]);
        }
        lmax = warp_best(lmax);

        float key[NT], sum = 0.f, pmax = 0.f;
        if (need_p || (!a.sigmoid && !a.renorm)) {
            if (a.sigmoid) {
#pragma unroll
                for (int j = 0; j < NT; j++)  // 0 for -inf
                    key[j] = route_sigmoid(l[j]);
            } else {
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    key[j] = l[j] > -INFINITY ? __expf(l[j] - lmax) : 0.f;
                    sum += key[j];
                }
                sum = warp_sum(sum);
                const float inv = 1.f / sum;
                pmax = inv;
#pragma unroll
                for (int j = 0; j < NT; j++)
                    key[j] *= inv;
            }
        }
        // Two fp32 keys closer than tol may be in the other order in 64 bits.  In half steps, p is off by 5 of its own
        // for the exponential, 2 |x| for the rounded argument x of it (p |x| is at most pmax max(1, -lmax)), 6 for
        // reciprocal and product, 20 for a softmax's sum of up to 512 terms in a tree; p + bias by one of the sum's.
        float tol_p = 0.f;
        if (need_p) {
            pmax = a.sigmoid ? route_sigmoid(lmax) : pmax;
            tol_p = 2.f * 5.97e-8f * ((a.sigmoid ? 12.f : 32.f) + 2.f * fmaxf(1.f, a.sigmoid ? -lmax : 1.f)) * pmax;
        }
        constexpr float HALF_STEP2 = 2.f * 5.97e-8f;
        bool sure = true;
        float group_best = 0.f, group_next = 0.f;  // of this lane's experts, by what scores groups
        if (by_logit) {
            if (need_p) {  // the two best p of the lane are those of its two best logits
                float b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const float v = l[j] > -INFINITY ? key[j] : -INFINITY;
                    b2 = v > b1 ? b1 : fmaxf(b2, v);
                    b1 = fmaxf(b1, v);
                }
                group_best = b1;
                group_next = b2;
                if (!lanes_of_group) {
#pragma unroll
                    for (int j = 0; j < NT; j++)
                        s_keys[e0 + j] = l[j] > -INFINITY ? key[j] : -INFINITY;
                }
            }
#pragma unroll
            for (int j = 0; j < NT; j++)
                key[j] = l[j];
        } else {
#pragma unroll
            for (int j = 0; j < NT; j++)
                key[j] = l[j] > -INFINITY ? key[j] + bias[j] : -INFINITY;
        }
        if (a.n_groups > 1 && !lanes_of_group && !(by_logit && need_p)) {
#pragma unroll
            for (int j = 0; j < NT; j++)
                s_keys[e0 + j] = key[j];
        }
        {
            int place[NT];
#pragma unroll
            for (int i = 0; i < LISTS; i++)
                places_of<LN>(key + i * LN, place + i * LN);
#pragma unroll
            for (int j = 0; j < NT; j++)
                sorted[j / LN * (LN + 1) + place[j]][lane] = make_float2(key[j], __int_as_float(e0 + j));
        }
        __syncwarp();

        if (a.n_groups > 1) {
            if (!by_logit || !need_p) {
                group_best = sorted[0][lane].x;
                group_next = sorted[1][lane].x;  // NT = 1: -inf
                if (LISTS > 1) {
                    const float ob = sorted[LN + 1][lane].x, on = sorted[LN + 2][lane].x;
                    group_next = fmaxf(fminf(group_best, ob), fmaxf(group_next, on));
                    group_best = fmaxf(group_best, ob);
                }
            }
            int g = lane;  // the group whose score this lane has
            if (lanes_of_group) {
                g = lane >> a.lane_shift;
                for (int o = 1; o < span; o <<= 1) {
                    const float ob = __shfl_xor_sync(0xffffffffu, group_best, o);
                    const float on = __shfl_xor_sync(0xffffffffu, group_next, o);
                    group_next = fmaxf(fminf(group_best, ob), fmaxf(group_next, on));
                    group_best = fmaxf(group_best, ob);
                }
            } else {
                group_best = group_next = -INFINITY;
                if (lane < a.n_groups)
                    for (int i = 0; i < gs; i++) {
                        const float v = (float)s_keys[lane * gs + i];  // exact: fp32 values
                        group_next = v > group_best ? group_best : fmaxf(group_next, v);
                        group_best = fmaxf(group_best, v);
                    }
            }
            // Keys are finite, but the sum of two may not be in fp32: such a group counts as the lowest or the largest, it is
            // not out, and the order of several of them is for 64 bits.
            const bool live = g < a.n_groups && group_best > -INFINITY;
            const float sum2 = a.group_top > 1 && group_next > -INFINITY ? group_best + group_next : group_best;
            const float score = live ? fmaxf(sum2, -FLT_MAX) : -INFINITY;
            // a group's place: the groups in front of it
            int place = 0;
            const int step = lanes_of_group ? span : 1;
            for (int i = 0; i < a.n_groups; i++) {
                const float o = __shfl_sync(0xffffffffu, score, i * step);
                place += o > score || (o == score && i < g);
            }
            const bool in = live && place < a.topk_groups;
            if (!(by_logit && a.group_top == 1) && a.topk_groups < a.n_groups) {
                const float low = -warp_best(in ? -score : -INFINITY);
                const float high = warp_best(!in && g < a.n_groups ? score : -INFINITY);
                // a score is off by its two keys' errors and a rounding; the keys may be far larger than their sum
                const float big = warp_best(fmaxf(group_best > -INFINITY ? fabsf(group_best) : 0.f,
                                                  group_next > -INFINITY ? fabsf(group_next) : 0.f));
                if (high > -INFINITY)
                    sure = low - high > 2.f * tol_p + 4.f * HALF_STEP2 * big;
            }
            if (lanes_of_group) {
                if (!in)
#pragma unroll
                    for (int i = 0; i < LISTS; i++)
                        sorted[i * (LN + 1)][lane].x = -INFINITY;
            } else {
                const unsigned kept = __ballot_sync(0xffffffffu, in);
#pragma unroll 1
                for (int i = 0; i < LISTS; i++) {
                    float2(*list)[32] = sorted + i * (LN + 1);
                    int n = 0;
#pragma unroll 1
                    for (int j = 0; j < LN; j++) {  // those that stay move up
                        const float2 v = list[j][lane];
                        const int e = __float_as_int(v.y);
                        if (v.x > -INFINITY && e < a.E && ((kept >> (e / gs)) & 1u))
                            list[n++][lane] = v;
                    }
                    for (int j = n; j < LN; j++)
                        list[j][lane].x = -INFINITY;
                }
            }
        }

        // Rounds: the largest head, of the lowest lane that has it; that lane leaves the expert in `sel` and
        // moves on.  Lane k keeps the key of round k.
        float2 head = sorted[0][lane];
        float mine_key = -INFINITY;
        const float2* next = &sorted[1][lane];
        float2 other = make_float2(-INFINITY, 0.f);  // the second list's head; `head` is the larger, the first list's in a tie
        const float2* other_next = nullptr;
        bool second = false;
        auto larger = [&]() {
            if (second ? other.x >= head.x : other.x > head.x) {
                const float2 h = head;
                const float2* n = next;
                head = other, next = other_next, other = h, other_next = n;
                second = !second;
            }
        };
        if (LISTS > 1) {
            other = sorted[LN + 1][lane];
            other_next = &sorted[LN + 2][lane];
            larger();
        }
        const unsigned lower = (1u << lane) - 1u;
        auto round = [&](int k) {
            const float top = warp_best(head.x);
            const unsigned has = __ballot_sync(0xffffffffu, head.x == top);
            if (lane == k)
                mine_key = top;
            if (head.x == top && top > -INFINITY && !(has & lower)) {  // a list ends with -inf
                sel[k] = __float_as_int(head.y);
                head = *next;
                next += 32;
                if (LISTS > 1)
                    larger();
            }
            return top;
        };
        const int rounds = by_logit ? a.K : a.K + 1;  // the first that is left out has a gap to keep too
#pragma unroll 1
        for (int k = 0; k < rounds; k++)
            round(k);
        bool close = false;
        float tol = 0.f;
        if (!by_logit) {
            const float before = __shfl_up_sync(0xffffffffu, mine_key, 1);
            tol = tol_p + HALF_STEP2 * fmaxf(fabsf(before), fabsf(mine_key));
            close = __any_sync(0xffffffffu, lane > 0 && lane < rounds && mine_key > -INFINITY && !(before - mine_key > tol));
        }
        __syncwarp();
        int mine = lane < a.K && mine_key > -INFINITY ? sel[lane] : -1;
        if (close && sure) {
            // Who may be among the K: everybody within tol of the K-th.  A lane each, in 64 bits, then their ranks.
            const float low = __shfl_sync(0xffffffffu, mine_key, a.K - 1);
            const float cut = low - (tol_p + HALF_STEP2 * fabsf(low));
            int n = __popc(__ballot_sync(0xffffffffu, mine_key > -INFINITY));
            bool more = n == rounds;
            while (more && n < 32) {
                const float top = round(n);
                more = top > -INFINITY && top >= cut;
                n += more;
            }
            __syncwarp();
            sure = !more;
            if (sure) {
                const int e = lane < n ? sel[lane] : 0;
                double full = 0.0;
                if (!a.sigmoid) {
#pragma unroll 1
                    for (int j = 0; j < have; j++) {
                        const float v = route_logit(load_as_float(a.logits, at + e0 + j, a.dtype));
                        if (v > -INFINITY)
                            full += exp((double)v - (double)lmax);
                    }
                    full = warp_sum(full);
                }
                double exact = -INFINITY;
                if (lane < n) {
                    const double v = route_logit(load_as_float(a.logits, at + e, a.dtype));
                    exact = (a.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - (double)lmax) / full) + (double)fminf(a.bias[e], FLT_MAX);
                }
                int rank = 0;
                for (int i = 0; i < n; i++) {
                    const double o = __shfl_sync(0xffffffffu, exact, i);
                    const int oe = __shfl_sync(0xffffffffu, e, i);
                    rank += o > exact || (o == exact && oe < e);
                }
                __syncwarp();
                if (lane < n)
                    sel[rank] = e;
                __syncwarp();
                mine = lane < a.K && lane < n ? sel[lane] : -1;
            }
        }
        if (!sure)
            mine = route_exact(a, t, lmax, s_keys, lane);

        // The weights, lane k that of slot k.  Where they are divided by their sum, the exponentials are taken
        // relative to the largest selected, so that weights far below the best expert keep their ratios:
        // sigmoid(x) = exp(min(x, 0)) / (1 + exp(-|x|)).
        float w = 0.f;
        const float x = mine >= 0 ? route_logit(load_as_float(a.logits, at + mine, a.dtype)) : -INFINITY;
        const float y = a.sigmoid ? fminf(x, 0.f) : x;
        const float ref = a.renorm ? warp_best(y) : a.sigmoid ? 0.f : lmax;
        if (mine >= 0) {
            const float d = y - ref;
            if (d > -104.f) {  // below, 0 in fp32
                const float back = (float)(((double)y - (double)ref) - (double)d);  // what rounding d left out
                w = expf(d);
                w = fmaf(w, back, w);
                if (a.sigmoid)
                    w = w / (1.f + expf(-fabsf(x)));
            }
        }
        if (a.renorm)
            sum = warp_sum(w);
        if (a.renorm || !a.sigmoid)
            w = w > 0.f ? w / sum : 0.f;  // sum: of the selected, or of the softmax
        if (lane < a.K) {
            a.topk_i[(size_t)t * a.K + lane] = mine;
            a.topk_w[(size_t)t * a.K + lane] = w * a.scale;
        }
        __syncwarp();
    }
}

// Slots per expert, from the indices; `counts` were cleared by the kernel in front.  256 tokens,
// 256 experts, top 8: 3.1 us without counts, 6.1 with, 6.8 launched the ordinary way, 7.7 counted in the routing
// kernel behind a fill; counted by one cluster with all tokens on its 8 SMs 7.7, with groups 13.8.
__global__ void __launch_bounds__(256) route_counts_kernel(const int* topk_i, int n, int E, int* counts) {
    __shared__ int s_hist[ROUTE_MAX_E];
    for (int i = threadIdx.x; i < E; i += blockDim.x)
        s_hist[i] = 0;
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) {
        const int e = topk_i[i];
        if (e >= 0)
            atomicAdd(&s_hist[e], 1);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < E; i += blockDim.x)
        if (s_hist[i])
            atomicAdd(&counts[i], s_hist[i]);
}

}  // namespace op
}  // namespace moe
