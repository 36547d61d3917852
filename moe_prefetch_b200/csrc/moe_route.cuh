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
// Ties go to the lower index, and a NaN counts as -inf, everywhere.  With `masked`
// an expert whose logit is -inf has c = -inf, and a group's sum leaves out -inf.
struct RouteSpec {
    int n_expert, k, sigmoid, n_group, topk_group, group_top, renorm, masked;
    int per;       // experts per group
    int log_lanes; // 2^log_lanes lanes per group: the largest power of two <= 32 / n_group
    float scale;
    const float *bias;   // [n_expert] or null
};

constexpr int ROUTE_MAX_EXPERT = 512;
constexpr int ROUTE_MAX_GROUP = 32;
constexpr int ROUTE_MAX_K = 32;

// The rule of checked arguments, with its derived fields.
inline RouteSpec route_spec(int n_expert, int k, int sigmoid, int n_group, int topk_group, int group_top, int renorm,
                            int masked, float scale, const float *bias) {
    RouteSpec s{n_expert, k, sigmoid, n_group, topk_group, group_top, renorm, masked, n_expert / n_group, 5, scale, bias};
    while (n_group << s.log_lanes > 32) --s.log_lanes;
    return s;
}
// Experts each lane holds.  At most 30 for ROUTE_MAX_EXPERT experts in up to
// ROUTE_MAX_GROUP groups (more than 16 of the 32 lanes have a group).
inline int route_per_lane(const RouteSpec &s) { return ((s.per - 1) >> s.log_lanes) + 1; }

// The lane layout: with q = 2^log_lanes, group g's experts go to lanes [g q,
// (g + 1) q), expert g * per + i + q j to lane g q + i as its j-th.  A group
// score is then a butterfly over q lanes; with one group it is the plain strided
// layout.
struct RouteLane {
    int group, first, step, count;   // experts first, first + step, ... (count of them)
    __device__ __forceinline__ RouteLane(const RouteSpec &s, int lane) {
        group = lane >> s.log_lanes;
        step = 1 << s.log_lanes;
        const int i = lane & (step - 1);
        first = group * s.per + i;
        count = group < s.n_group && i < s.per ? ((s.per - 1 - i) >> s.log_lanes) + 1 : 0;
    }
    __device__ __forceinline__ int expert(int j) const { return first + step * j; }
};

// A choice value as it is compared: NaN counts as -inf, -0 as +0.
__device__ __forceinline__ float route_clean(float v) { return isnan(v) ? -INFINITY : v + 0.0f; }
__device__ __forceinline__ double route_clean(double v) { return isnan(v) ? -(double)INFINITY : v + 0.0; }

// Order-preserving integer keys of clean values, all > 0 (0 is free for "none").
__device__ __forceinline__ uint32_t route_key(float v) {
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t route_key(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
// Largest value of the warp, by shuffles.
__device__ __forceinline__ float route_warp_max(float v) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor_sync(MOE_FULL, v, off));
    return v;
}

// The score of this lane's group: the largest clean value, or with group_top 2
// the sum of the two largest.
template <typename V, int J>
__device__ __forceinline__ V route_group(const V (&c)[J], int count, const RouteSpec &s) {
    V b1 = -(V)INFINITY, b2 = b1;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const V v = j < count ? c[j] : -(V)INFINITY;
        b2 = max(b2, min(b1, v));
        b1 = max(b1, v);
    }
    for (int off = 1; off < 1 << s.log_lanes; off <<= 1) {
        const V o1 = __shfl_xor_sync(MOE_FULL, b1, off), o2 = __shfl_xor_sync(MOE_FULL, b2, off);
        b2 = max(min(b1, o1), max(b2, o2));
        b1 = max(b1, o1);
    }
    return route_clean(s.group_top == 2 && s.per > 1 && !(s.masked && b2 == -(V)INFINITY) ? b1 + b2 : b1);
}

// True when this lane's group (its key gk, the same in all its lanes) is among
// the topk_group largest.
template <typename K>
__device__ __forceinline__ bool route_group_kept(const RouteSpec &s, K gk, int group) {
    int before = 0;
    for (int o = 0; o < s.n_group; ++o) {
        const K ok = __shfl_sync(MOE_FULL, gk, o << s.log_lanes);
        before += ok > gk || (ok == gk && o < group) ? 1 : 0;
    }
    return before < s.topk_group;
}

// (key, j) before (okey, oj): the larger key, then the lower j
__device__ __forceinline__ void route_cx(uint32_t &ka, int &ja, uint32_t &kb, int &jb) {
    const bool swap = kb > ka || (kb == ka && jb < ja);
    const uint32_t k = swap ? kb : ka;
    const int j = swap ? jb : ja;
    kb = swap ? ka : kb;
    jb = swap ? ja : jb;
    ka = k;
    ja = j;
}

// Batcher's odd-even merge sort of a lane's J keys, largest first; cx(i, j) orders
// entries i < j.
template <int J, typename CX>
__device__ __forceinline__ void route_sort(CX cx) {
#pragma unroll
    for (int p = 1; p < J; p *= 2)
#pragma unroll
        for (int q = p; q >= 1; q /= 2)
#pragma unroll
            for (int j = q % p; j <= J - 1 - q; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; ++i)
                    if (i + j + q < J && (i + j) / (2 * p) == (i + j + q) / (2 * p)) cx(i + j, i + j + q);
}

// The k largest keys (0: none) of the warp in order: returns rank r's expert in
// lane r < k.  Up to eight keys per lane are sorted first, so that a round looks
// at one key per lane; more are searched every round.
template <int J>
__device__ __forceinline__ int route_topk(uint32_t (&key)[J], const RouteSpec &s, const RouteLane &me, int lane) {
    constexpr bool SORT = J <= 8;
    int at[J];
#pragma unroll
    for (int j = 0; j < J; ++j) at[j] = j;
    if constexpr (SORT) route_sort<J>([&](int i, int j) { route_cx(key[i], at[i], key[j], at[j]); });
    int id_r = 0;
    for (int r = 0; r < s.k; ++r) {
        uint32_t best = key[0];
        int bj = at[0];
        if constexpr (!SORT) {
#pragma unroll
            for (int j = 1; j < J; ++j)
                if (key[j] > best) { best = key[j]; bj = j; }
        }
        const uint32_t m = __reduce_max_sync(MOE_FULL, best);
        const int id = (int)__reduce_min_sync(MOE_FULL, best == m ? (unsigned)me.expert(bj) : (unsigned)ROUTE_MAX_EXPERT);
        const bool mine = best == m && me.expert(bj) == id;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if constexpr (SORT) {   // the list moves up
                key[j] = mine ? j + 1 < J ? key[j + 1 < J ? j + 1 : j] : 0u : key[j];
                at[j] = mine && j + 1 < J ? at[j + 1 < J ? j + 1 : j] : at[j];
            } else {
                key[j] = mine && j == bj ? 0u : key[j];
            }
        }
        if (lane == r) id_r = id;
    }
    return id_r;
}

// The same for keys that carry their place: value * 32 + (31 - j), so that a
// comparison orders both at once and the sort is two instructions a pair.  The
// first k + 1 are compared, and -1 is returned when two neighbours are within
// tol of each other.
template <int J>
__device__ __forceinline__ int route_topk_packed(uint32_t (&key)[J], const RouteSpec &s, const RouteLane &me, int lane,
                                                 uint32_t tol) {
    constexpr bool SORT = J <= 8;
    if constexpr (SORT)
        route_sort<J>([&](int i, int j) {
            const uint32_t hi = max(key[i], key[j]);
            key[j] = min(key[i], key[j]);
            key[i] = hi;
        });
    uint32_t last = 0xffffffffu;
    int id_r = 0;
    for (int r = 0; r <= s.k; ++r) {
        uint32_t best = key[0];
        if constexpr (!SORT) {
#pragma unroll
            for (int j = 1; j < J; ++j) best = max(best, key[j]);
        }
        const uint32_t m = __reduce_max_sync(MOE_FULL, best);
        if (r && m && last - m <= tol) return -1;   // (m = 0: no expert is left to be confused with)
        if (r == s.k) break;
        last = m;
        // of lanes with the same key only one moves on: the next round then sees the tie
        const int owner = __ffs(__ballot_sync(MOE_FULL, best == m)) - 1;
        const bool mine = lane == owner;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if constexpr (SORT) key[j] = mine ? j + 1 < J ? key[j + 1 < J ? j + 1 : j] : 0u : key[j];
            else key[j] = mine && key[j] == m ? 0u : key[j];
        }
        const int id = __shfl_sync(MOE_FULL, me.expert(31 - (int)(m & 31)), owner);
        if (lane == r) id_r = id;
    }
    return id_r;
}

// The same for 64-bit values of the lanes' `alive` experts.
template <int J>
__device__ __forceinline__ int route_topk(const double (&c)[J], uint32_t alive, const RouteSpec &s, const RouteLane &me,
                                          int lane) {
    int id_r = 0;
    for (int r = 0; r < s.k; ++r) {
        double best = 0.0;
        int bj = -1;
#pragma unroll
        for (int j = 0; j < J; ++j)
            if ((alive >> j & 1) && (bj < 0 || c[j] > best)) { best = c[j]; bj = j; }
        const uint64_t k = bj < 0 ? 0ull : route_key(best);
        const uint32_t hi = __reduce_max_sync(MOE_FULL, (uint32_t)(k >> 32));
        const uint32_t lo = __reduce_max_sync(MOE_FULL, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
        const bool top = k && k == ((uint64_t)hi << 32 | lo);
        const int id = (int)__reduce_min_sync(MOE_FULL, top ? (unsigned)me.expert(bj) : (unsigned)ROUTE_MAX_EXPERT);
        if (top && me.expert(bj) == id) alive &= ~(1u << bj);
        if (lane == r) id_r = id;
    }
    return id_r;
}

// Selection by 32-bit choice values where their rounding cannot matter: -1 when
// some value is not finite, or two neighbours among the first k + 1, or the last
// kept and first dropped group, are closer than twice their error.  With u =
// 2^-24, the error of a value c is at most 10 u max(1, |c|) for sigmoid (expf 4 u
// of a value below 1, a division of 4 u, two additions) and 30 u max(1, |c|) for
// softmax (the sum's up to 15 additions, too): 2^-20 and 2^-18 are taken.  A
// sum of two has twice that and its own rounding.  The values are then compared
// as integers of 26 bits below the largest, with an error of 2^-26 more.
template <int J>
__device__ __forceinline__ int route_fast(const float (&l)[J], const RouteSpec &s, const RouteLane &me, float mx, int lane,
                                          float &total) {
    float c[J], b[J], sum[4] = {0.0f, 0.0f, 0.0f, 0.0f}, big = 1.0f, odd = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j) b[j] = s.bias && j < me.count ? s.bias[me.expert(j)] : 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j) c[j] = expf(s.sigmoid ? -l[j] : l[j] - mx);   // (a lane without a j-th expert: inf or 0)
    if (s.sigmoid) {
#pragma unroll
        for (int j = 0; j < J; ++j) c[j] = __fdividef(1.0f, 1.0f + c[j]) + b[j];
    } else {
#pragma unroll
        for (int j = 0; j < J; ++j) sum[j & 3] += c[j];
        total = warp_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
        const float inv = 1.0f / total;
#pragma unroll
        for (int j = 0; j < J; ++j) c[j] = fmaf(c[j], inv, b[j]);
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
        big = fmaxf(big, fabsf(c[j]));
        odd = fmaf(c[j], 0.0f, odd);   // NaN once some value is not finite
    }
    if (!__all_sync(MOE_FULL, odd == 0.0f)) return -1;
    big = route_warp_max(big);
    const float err = big * (s.sigmoid ? 0x1p-20f : 0x1p-18f);
    bool kept = true;
    if (s.n_group > 1) {
        const bool mine = me.group < s.n_group;
        const float g = route_group(c, me.count, s);
        kept = route_group_kept(s, route_key(g), me.group);
        const float lo = -route_warp_max(mine && kept ? -g : -INFINITY);   // the smallest kept
        const float hi = route_warp_max(mine && !kept ? g : -INFINITY);    // the largest left out, if any
        if (lo - hi <= 6.0f * err) return -1;
    }
    // scaled by a power of two so that |c| <= 2^25
    const uint32_t two = (__float_as_uint(big) + 0x7fffffu) & 0x7f800000u;   // big, rounded up to a power of two
    if (two == 0x7f800000u) return -1;
    const float scale = __uint_as_float(((127u + 25u + 127u) << 23) - two);
    uint32_t key[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int q = __float2int_rn(c[j] * scale) + (1 << 25) + 1;   // 1 .. 2^26 + 1
        key[j] = kept && j < me.count ? (uint32_t)q * 32u + (31u - j) : 0u;
    }
    return route_topk_packed(key, s, me, lane, (uint32_t)__float2int_ru(2.0f * err * scale + 1.0f) * 32u + 31u);
}

// Selection by 64-bit values, which a softmax with a NaN or +inf logit (bad)
// makes NaN; with `prior`, delta is added to the experts that are resident
// (prior_resident), after the groups.
template <int J>
__device__ __forceinline__ int route_exact(const float (&l)[J], const RouteSpec &s, const RouteLane &me, float mx, bool bad,
                                           const int32_t *table, int ns, float delta, bool prior, const int32_t *pub,
                                           int lane) {
    double c[J], total = 0.0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        c[j] = 0.0;
        if (j >= me.count) continue;
        c[j] = s.sigmoid ? 1.0 / (1.0 + exp(-(double)l[j])) : mx > -INFINITY ? exp((double)l[j] - (double)mx) : 0.0;
        total += c[j];
    }
    double inv = 1.0;
    if (!s.sigmoid) {
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) total += __shfl_xor_sync(MOE_FULL, total, off);
        inv = bad ? NAN : total == 0.0 ? 0.0 : 1.0 / total;
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
        if (j < me.count) {
            c[j] = route_clean(c[j] * inv + (s.bias ? (double)s.bias[me.expert(j)] : 0.0));
            if (s.masked && l[j] == -INFINITY) c[j] = -(double)INFINITY;
        }
    const bool kept = s.n_group == 1 || route_group_kept(s, route_key(route_group(c, me.count, s)), me.group);
    uint32_t alive = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        if (!kept || j >= me.count) continue;
        alive |= 1u << j;
        if (prior && prior_resident(table, ns, pub, me.expert(j))) c[j] += (double)delta;
    }
    return route_topk(c, alive, s, me, lane);
}

__device__ __forceinline__ float route_load(const float *p) { return *p; }
__device__ __forceinline__ float route_load(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ float route_load(const __half *p) { return __half2float(*p); }

// One token's ids and weights (lane r < k gets rank r's) from its logits in
// shared or global memory, at most J per lane.
//
// Without bias and prior the choice values fall with the logits, which are
// compared as they are.  Otherwise 32-bit scores decide where they are far
// enough apart (route_fast: about 998 tokens in 1000), and 64-bit scores where
// their rounding could decide between two experts, and for tokens with masked
// experts.
//
// The weights are formed in 32 bits (expf 4 u with the rounding of l - mx taken
// back, k - 1 additions in five levels, two divisions, scale: below 20 u);
// renormalised ones in 64 bits where a score underflows or their sum is very small.
template <int J, typename T>
__device__ __forceinline__ void route_warp_row(const T *row, const RouteSpec &s, const int32_t *table, int ns,
                                               float delta, bool prior, const int32_t *pub, int lane, int &id_r,
                                               float &w_r) {
    static_assert(J <= 32, "one bit of a mask per expert of a lane");
    const RouteLane me(s, lane);
    float l[J], mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < J; ++j) l[j] = j < me.count ? route_load(row + me.expert(j)) : -INFINITY;
    if (!s.sigmoid) {
#pragma unroll
        for (int j = 0; j < J; ++j) mx = fmaxf(mx, l[j]);
        mx = route_warp_max(mx);
    }
    // a NaN, or for softmax +inf: then every softmax score is NaN
    auto is_bad = [&]() {
        bool bad = false;
#pragma unroll
        for (int j = 0; j < J; ++j) bad = bad || isnan(l[j]);
        return __any_sync(MOE_FULL, bad) || mx == INFINITY;
    };
    bool bad = false;
    float total = 0.0f;   // of e^(l - mx) over all experts
    if (!s.bias && !prior && (s.n_group == 1 || s.group_top == 1)) {
        uint32_t key[J];
        bool kept = true;
        if (s.n_group > 1) {
            float c[J];
#pragma unroll
            for (int j = 0; j < J; ++j) c[j] = route_clean(l[j]);
            kept = route_group_kept(s, route_key(route_group(c, me.count, s)), me.group);
        }
#pragma unroll
        for (int j = 0; j < J; ++j) key[j] = kept && j < me.count ? route_key(route_clean(l[j])) : 0u;
        id_r = route_topk(key, s, me, lane);
        bad = !s.sigmoid && is_bad();
    } else {
        bool exact = prior;
        if (s.masked) {
            bool off = false;
#pragma unroll
            for (int j = 0; j < J; ++j) off = off || (j < me.count && l[j] == -INFINITY);
            exact = __any_sync(MOE_FULL, off) || prior;
        }
        id_r = exact ? -1 : route_fast<J>(l, s, me, mx, lane, total);   // (no bad logits where it succeeds)
        if (__any_sync(MOE_FULL, id_r < 0)) {
            bad = is_bad();
            id_r = route_exact<J>(l, s, me, mx, bad, table, ns, delta, prior, pub, lane);
        }
    }
    if (!s.sigmoid && !s.renorm) {
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < J; ++j) sum[j & 3] += j < me.count && mx > -INFINITY ? expf(l[j] - mx) : 0.0f;
        total = warp_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
    }
    const float l_r = lane < s.k ? route_load(row + id_r) : -INFINITY;
    float v = 0.0f;
    if (s.sigmoid) v = lane < s.k ? 1.0f / (1.0f + expf(-l_r)) : 0.0f;
    else if (bad) v = NAN;
    else if (mx > -INFINITY && l_r > -INFINITY) {
        const float d = l_r - mx, t = d - l_r;              // l_r - mx = d + rest exactly
        const float rest = (l_r - (d - t)) - (mx + t);
        v = expf(d);
        if (v > 0.0f) v = fmaf(v, rest, v);                 // (d may be -inf)
    }
    if (s.renorm) total = warp_sum(lane < s.k ? v : 0.0f);
    // a score other than 0 below fp32's normal range: its share of a small sum may not be small
    const bool low = __any_sync(MOE_FULL, v < 0x1p-126f && l_r > -INFINITY);
    if (low && s.sigmoid && !s.renorm && l_r < -80.0f) v = expf(l_r);   // (e^80 may be too large, 1 + e^-80 is 1)
    if (s.renorm && (low || total < 1e-20f)) {
        double x = 0.0, sum;
        if (lane < s.k)
            x = s.sigmoid ? 1.0 / (1.0 + exp(-(double)l_r)) : mx > -INFINITY ? exp((double)l_r - (double)mx) : 0.0;
        sum = x;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(MOE_FULL, sum, off);
        v = sum == 0.0 ? 0.0f : (float)(x / sum);
    } else if (s.renorm || !s.sigmoid) {
        v = total == 0.0f && !bad ? 0.0f : v / total;   // (bad, softmax: v is NaN, and total may be 0 beside it)
    }
    w_r = v * s.scale;
}

}  // namespace moe
