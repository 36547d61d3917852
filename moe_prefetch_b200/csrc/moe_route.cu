// moe_route.cu -- expert routing from logits (moe_route), one warp per token.
#include "moe_kernels.h"

namespace moe {

#define ROUTE_WARPS 4

// grid ceil(n_tok / ROUTE_WARPS); block ROUTE_WARPS warps.  A warp per token: a
// token's experts fit its lanes' registers, and no barrier is needed.  Bound by
// integer instructions (the ALU pipe is 64 % busy): 8,192 tokens of 256 experts in
// four groups, sigmoid and bias, bf16, take 15.3 us (0.7 us of memory traffic);
// one token of 128 experts takes 2.2 us, the launch included.
template <typename T, int J>
__global__ void __launch_bounds__(ROUTE_WARPS * 32)
    k_route(RouteSpec spec, const T *__restrict__ logits, int64_t ld, int n_tok, int32_t *__restrict__ ids,
            float *__restrict__ w) {
    pdl_enter();
    const int lane = threadIdx.x & 31;
    const int t = blockIdx.x * ROUTE_WARPS + (threadIdx.x >> 5);
    if (t >= n_tok) return;
    int id_r;
    float w_r;
    route_warp_row<J>(logits + (int64_t)t * ld, spec, nullptr, 0, 0.0f, false, nullptr, lane, id_r, w_r);
    if (lane < spec.k) {
        ids[(size_t)t * spec.k + lane] = id_r;
        w[(size_t)t * spec.k + lane] = w_r;
    }
}

// One token of a layer, one warp: with the cache prior, and observed by one
// thread as the fused routers do.
__global__ void __launch_bounds__(32)
    k_route_one(RouteSpec spec, const float *__restrict__ logits, int32_t *__restrict__ ids, float *__restrict__ w,
                const int32_t *__restrict__ table, int ns, float delta, int use_prior, SlotState st,
                int observe_layer_idx, const int32_t *__restrict__ pub) {
    __shared__ int32_t sids[ROUTE_MAX_K];
    const int lane = threadIdx.x;
    int id_r;
    float w_r;
    route_warp_row<8>(logits, spec, table, ns, delta, use_prior != 0, pub, lane, id_r, w_r);
    if (lane < spec.k) {
        ids[lane] = sids[lane] = id_r;
        w[lane] = w_r;
    }
    __syncwarp();
    if (lane == 0) observe_layer(st, observe_layer_idx, sids, spec.k);
}

template <typename T>
static cudaError_t route_j(const RouteSpec &sp, const T *logits, int64_t ld, int n_tok, int32_t *ids, float *w,
                           cudaStream_t s) {
    const int grid = (n_tok - 1) / ROUTE_WARPS + 1;
    const int j = route_per_lane(sp);
    if (j <= 2) return launch_pdl(k_route<T, 2>, grid, ROUTE_WARPS * 32, 0, s, 0, sp, logits, ld, n_tok, ids, w);
    if (j <= 4) return launch_pdl(k_route<T, 4>, grid, ROUTE_WARPS * 32, 0, s, 0, sp, logits, ld, n_tok, ids, w);
    if (j <= 8) return launch_pdl(k_route<T, 8>, grid, ROUTE_WARPS * 32, 0, s, 0, sp, logits, ld, n_tok, ids, w);
    if (j <= 16) return launch_pdl(k_route<T, 16>, grid, ROUTE_WARPS * 32, 0, s, 0, sp, logits, ld, n_tok, ids, w);
    return launch_pdl(k_route<T, 32>, grid, ROUTE_WARPS * 32, 0, s, 0, sp, logits, ld, n_tok, ids, w);
}

cudaError_t launch_route(const RouteSpec &sp, const void *logits, int dtype, int64_t ld, int n_tok, int32_t *ids,
                         float *w, cudaStream_t s) {
    if (dtype == DT_BF16) return route_j(sp, (const __nv_bfloat16 *)logits, ld, n_tok, ids, w, s);
    if (dtype == DT_F16) return route_j(sp, (const __half *)logits, ld, n_tok, ids, w, s);
    return route_j(sp, (const float *)logits, ld, n_tok, ids, w, s);
}

cudaError_t launch_route_one(const RouteSpec &sp, const float *logits, int32_t *ids, float *w, const int32_t *table,
                             int ns, float delta, int use_prior, const SlotState &st, int observe_layer_idx,
                             const int32_t *pub, cudaStream_t s) {
    // a context has 32, 64, 128 or 256 experts: at most 8 per lane, whatever the groups
    if (route_per_lane(sp) > 8) return cudaErrorInvalidValue;
    k_route_one<<<1, 32, 0, s>>>(sp, logits, ids, w, table, ns, delta, use_prior, st, observe_layer_idx, pub);
    return cudaGetLastError();
}

}  // namespace moe
