// moe_route.cuh -- expert selection with a routing rule: softmax or sigmoid
// scores, a bias for balance, expert groups, top-k, renormalised and scaled
// weights.  One warp selects for one token; used by k_route (moe_route.cu) and
// by the batch router of a layer (moe_kernels.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "moe_dev.cuh"

namespace moe {

// A routing rule (moe_route_cfg with the derived fields).  With scores s and
// choice values c = s + bias:
//   groups: of n_group groups of `per` consecutive experts, the topk_group
//           with the largest group score (the largest c, or the sum of the two
//           largest) keep their experts;
//   ids:    the k largest c of the kept experts, in order;
//   w:      s[ids] (divided by their sum), times scale.
// Ties go to the lower index, and a NaN counts as -inf, everywhere.
struct RouteSpec {
    int n_expert, k, sigmoid, n_group, topk_group, group_top, renorm;
    int per;       // experts per group
    int lanes;     // lanes per group: the largest power of two <= 32 / n_group
    float scale;
    const float *bias;   // [n_expert] or null
};

constexpr int ROUTE_MAX_EXPERT = 512;
constexpr int ROUTE_MAX_GROUP = 32;
constexpr int ROUTE_MAX_K = 32;

// The rule of checked arguments, with its derived fields.
inline RouteSpec route_spec(int n_expert, int k, int sigmoid, int n_group, int topk_group, int group_top, int renorm,
                            float scale, const float *bias) {
    RouteSpec s{n_expert, k, sigmoid, n_group, topk_group, group_top, renorm, n_expert / n_group, 32, scale, bias};
    while (s.lanes * n_group > 32) s.lanes >>= 1;
    return s;
}
// Experts each lane holds: per / lanes rounded up.  At most 30 for
// ROUTE_MAX_EXPERT experts in up to ROUTE_MAX_GROUP groups (lanes * n_group
// > 16).
inline int route_per_lane(const RouteSpec &s) { return (s.per + s.lanes - 1) / s.lanes; }

// The lane layout: group g's experts go to lanes [g * lanes, (g + 1) * lanes),
// expert g * per + i + lanes * j to lane g * lanes + i as its j-th.  A group
// score is then a butterfly over `lanes` lanes; with one group it is the plain
// strided layout.  -1: the lane has no j-th expert.
__device__ __forceinline__ int route_expert(const RouteSpec &s, int lane, int j) {
    const int g = lane / s.lanes, i = (lane & (s.lanes - 1)) + s.lanes * j;
    return g < s.n_group && i < s.per ? g * s.per + i : -1;
}

// Order-preserving integer keys, all > 0 (0 is free for "no expert"); NaN
// counts as -inf, -0 as +0.
__device__ __forceinline__ uint32_t route_key(float v) {
    v = isnan(v) ? -INFINITY : v + 0.0f;
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t route_key(double v) {
    v = isnan(v) ? -(double)INFINITY : v + 0.0;
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

__device__ __forceinline__ uint32_t route_max(uint32_t v) { return __reduce_max_sync(MOE_FULL, v); }
__device__ __forceinline__ uint64_t route_max(uint64_t v) {
    const uint32_t hi = __reduce_max_sync(MOE_FULL, (uint32_t)(v >> 32));
    const uint32_t lo = __reduce_max_sync(MOE_FULL, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
    return (uint64_t)hi << 32 | lo;
}

// True when this lane's group (its key gk, the same in all its lanes) is among
// the topk_group largest.
template <typename K>
__device__ __forceinline__ bool route_group_kept(const RouteSpec &s, K gk, int lane) {
    const int g = lane / s.lanes;
    int before = 0;
    for (int o = 0; o < s.n_group; ++o) {
        const K ok = __shfl_sync(MOE_FULL, gk, o * s.lanes);
        before += ok > gk || (ok == gk && o < g) ? 1 : 0;
    }
    return before < s.topk_group;
}

// The k largest keys (0: not to be chosen) of the warp in order: lane r < k
// gets the id of rank r and that expert's logit.
template <typename K, int J>
__device__ __forceinline__ void route_topk(const K (&key)[J], const float (&l)[J], const RouteSpec &s, int lane,
                                           int &id_r, float &l_r) {
    uint32_t taken = 0;
    for (int r = 0; r < s.k; ++r) {
        K best = 0;
        float bl = 0.0f;
        int bj = 0;
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (!(taken >> j & 1) && key[j] > best) { best = key[j]; bl = l[j]; bj = j; }
        const K m = route_max(best);
        const int e = best == m && m ? route_expert(s, lane, bj) : ROUTE_MAX_EXPERT;
        const int id = (int)__reduce_min_sync(MOE_FULL, (unsigned)e);
        const int owner = __ffs(__ballot_sync(MOE_FULL, e == id)) - 1;
        if (lane == owner) taken |= 1u << bj;
        bl = __shfl_sync(MOE_FULL, bl, owner);
        if (lane == r) { id_r = id; l_r = bl; }
    }
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(MOE_FULL, v, off);
    return v;
}

// One token: l[j] the logit of expert route_expert(s, lane, j).  Lane r < k
// gets rank r's id and weight.  With `prior`, delta is added to the choice
// value of the experts that are resident (prior_resident), after the groups.
//
// Without bias and prior the choice values fall with the logits, which are
// compared as they are.  Otherwise the scores are computed and compared in 64
// bits: in 32 bits the rounding of 1 / (1 + e^-l) would decide between close
// experts.  The weights are formed in 64 bits, once per chosen expert.
template <int J>
__device__ __forceinline__ void route_warp(const float (&l)[J], const RouteSpec &s, const int32_t *table, int ns,
                                           float delta, bool prior, const int32_t *pub, int lane, int &id_r,
                                           float &w_r) {
    static_assert(J <= 32, "one bit of a mask per expert of a lane");
    float mx = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int j = 0; j < J; ++j)
        if (route_expert(s, lane, j) >= 0) {
            nan |= isnan(l[j]);
            mx = fmaxf(mx, l[j]);
        }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(MOE_FULL, mx, off));
    nan = __any_sync(MOE_FULL, nan) || mx == INFINITY;   // then every softmax score is NaN
    double total = 0.0;   // of e^(l - mx) over all experts, where it is needed
    float l_r = 0.0f;
    id_r = 0;
    if (!s.bias && !prior && (s.n_group == 1 || s.group_top == 1)) {
        uint32_t key[J];
#pragma unroll
        for (int j = 0; j < J; ++j) key[j] = route_expert(s, lane, j) >= 0 ? route_key(l[j]) : 0u;
        if (s.n_group > 1) {
            uint32_t gk = 0;
#pragma unroll
            for (int j = 0; j < J; ++j) gk = max(gk, key[j]);
            for (int off = 1; off < s.lanes; off <<= 1) gk = max(gk, __shfl_xor_sync(MOE_FULL, gk, off));
            if (!route_group_kept(s, gk, lane)) {
#pragma unroll
                for (int j = 0; j < J; ++j) key[j] = 0u;
            }
        }
        route_topk(key, l, s, lane, id_r, l_r);
        if (!s.sigmoid && !s.renorm) {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (route_expert(s, lane, j) >= 0 && mx > -INFINITY) sum += expf(l[j] - mx);
            total = warp_sum_f64((double)sum);
        }
    } else {
        double c[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            c[j] = 0.0;
            if (route_expert(s, lane, j) < 0) continue;
            c[j] = s.sigmoid ? 1.0 / (1.0 + exp(-(double)l[j])) : mx > -INFINITY ? exp((double)l[j] - (double)mx) : 0.0;
            total += c[j];
        }
        if (!s.sigmoid) {
            total = warp_sum_f64(total);
            const double inv = total == 0.0 ? 0.0 : 1.0 / total;
#pragma unroll
            for (int j = 0; j < J; ++j) c[j] = nan ? NAN : c[j] * inv;
        }
        uint64_t key[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int e = route_expert(s, lane, j);
            if (s.bias && e >= 0) c[j] += (double)s.bias[e];
            key[j] = e >= 0 ? route_key(c[j]) : 0ull;
        }
        if (s.n_group > 1) {
            double b1 = -(double)INFINITY, b2 = b1;   // the two largest of the group
#pragma unroll
            for (int j = 0; j < J; ++j) {
                if (route_expert(s, lane, j) < 0) continue;
                const double v = isnan(c[j]) ? -(double)INFINITY : c[j];
                b2 = fmax(b2, fmin(b1, v));
                b1 = fmax(b1, v);
            }
            for (int off = 1; off < s.lanes; off <<= 1) {
                const double o1 = __shfl_xor_sync(MOE_FULL, b1, off), o2 = __shfl_xor_sync(MOE_FULL, b2, off);
                b2 = fmax(fmin(b1, o1), fmax(b2, o2));
                b1 = fmax(b1, o1);
            }
            if (!route_group_kept(s, route_key(s.group_top == 2 && s.per > 1 ? b1 + b2 : b1), lane)) {
#pragma unroll
                for (int j = 0; j < J; ++j) key[j] = 0ull;
            }
        }
        if (prior) {
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int e = route_expert(s, lane, j);
                if (key[j] && prior_resident(table, ns, pub, e)) key[j] = route_key(c[j] + (double)delta);
            }
        }
        route_topk(key, l, s, lane, id_r, l_r);
    }
    double v = 0.0;
    if (lane < s.k) {
        if (s.sigmoid) v = 1.0 / (1.0 + exp(-(double)l_r));
        else if (nan) v = NAN;
        else if (mx > -INFINITY) v = exp((double)l_r - (double)mx);
    }
    if (s.renorm) total = warp_sum_f64(v);
    if (s.renorm || !s.sigmoid) v = total == 0.0 ? 0.0 : v / total;
    w_r = (float)(v * (double)s.scale);
}

__device__ __forceinline__ float route_load(const float *p) { return *p; }
__device__ __forceinline__ float route_load(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ float route_load(const __half *p) { return __half2float(*p); }

// route_warp over a token's logits in memory (shared or global).
template <int J, typename T>
__device__ __forceinline__ void route_warp_row(const T *row, const RouteSpec &s, const int32_t *table, int ns,
                                               float delta, bool prior, const int32_t *pub, int lane, int &id_r,
                                               float &w_r) {
    float l[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int e = route_expert(s, lane, j);
        l[j] = e >= 0 ? route_load(row + e) : 0.0f;
    }
    route_warp<J>(l, s, table, ns, delta, prior, pub, lane, id_r, w_r);
}

}  // namespace moe
