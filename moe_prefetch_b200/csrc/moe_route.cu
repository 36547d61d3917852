// moe_route.cu -- expert routing from logits (moe_route), one warp per token.
#include "moe_kernels.h"

namespace moe {

#define ROUTE_WARPS 4

// grid ceil(n_tok / ROUTE_WARPS); block ROUTE_WARPS warps.  With st the single
// token's layer is observed by one thread, as the fused routers do.
template <typename T, int J>
__global__ void __launch_bounds__(ROUTE_WARPS * 32)
    k_route(RouteSpec spec, const T *__restrict__ logits, int64_t ld, int n_tok, int32_t *__restrict__ ids,
            float *__restrict__ w, const int32_t *__restrict__ table, int ns, float delta, int use_prior,
            SlotState st, int observe_layer_idx, const int32_t *__restrict__ pub) {
    __shared__ int32_t sids[ROUTE_MAX_K];
    const int lane = threadIdx.x & 31;
    const int t = blockIdx.x * ROUTE_WARPS + (threadIdx.x >> 5);
    if (t >= n_tok) return;
    int id_r;
    float w_r;
    route_warp_row<J>(logits + (int64_t)t * ld, spec, table, ns, delta, use_prior != 0, pub, lane, id_r, w_r);
    if (lane < spec.k) {
        ids[(size_t)t * spec.k + lane] = id_r;
        w[(size_t)t * spec.k + lane] = w_r;
    }
    if (observe_layer_idx >= 0) {   // n_tok == 1: warp 0 only
        if (lane < spec.k) sids[lane] = id_r;
        __syncwarp();
        if (lane == 0) observe_layer(st, observe_layer_idx, sids, spec.k);
    }
}

template <typename T>
static cudaError_t route_j(const RouteSpec &sp, const T *logits, int64_t ld, int n_tok, int32_t *ids, float *w,
                           const int32_t *table, int ns, float delta, int use_prior, const SlotState &st, int obs,
                           const int32_t *pub, cudaStream_t s) {
    const int grid = (n_tok + ROUTE_WARPS - 1) / ROUTE_WARPS;
    const int j = route_per_lane(sp);
#define ROUTE_GO(J)                                                                                          \
    k_route<T, J><<<grid, ROUTE_WARPS * 32, 0, s>>>(sp, logits, ld, n_tok, ids, w, table, ns, delta,         \
                                                    use_prior, st, obs, pub)
    if (j <= 2) ROUTE_GO(2);
    else if (j <= 4) ROUTE_GO(4);
    else if (j <= 8) ROUTE_GO(8);
    else if (j <= 16) ROUTE_GO(16);
    else ROUTE_GO(32);
#undef ROUTE_GO
    return cudaGetLastError();
}

cudaError_t launch_route(const RouteSpec &sp, const void *logits, int dtype, int64_t ld, int n_tok, int32_t *ids,
                         float *w, const int32_t *table, int ns, float delta, int use_prior, const SlotState *st,
                         int observe_layer_idx, const int32_t *pub, cudaStream_t s) {
    const SlotState sst = st ? *st : SlotState{};
    const int obs = st ? observe_layer_idx : -1;
    if (dtype == DT_BF16)
        return route_j(sp, (const __nv_bfloat16 *)logits, ld, n_tok, ids, w, table, ns, delta, use_prior, sst, obs,
                       pub, s);
    if (dtype == DT_F16)
        return route_j(sp, (const __half *)logits, ld, n_tok, ids, w, table, ns, delta, use_prior, sst, obs, pub, s);
    return route_j(sp, (const float *)logits, ld, n_tok, ids, w, table, ns, delta, use_prior, sst, obs, pub, s);
}

}  // namespace moe
