// moe_adapters.cu -- low-rank adapters of many requests beside one projection:
//
//   out[t] = y[t] + scale[a] * B[a] (A[a] x[t]),   a = ids[t]
//
// with A [rank][n_in] and B [n_out][rank] in 16 bits.  The low-rank vector
// A x stays in fp32 between the two products.
#include "moe_kernels.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace moe {

__device__ __forceinline__ float ad_f32(float v) { return v; }
__device__ __forceinline__ float ad_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float ad_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void ad_store(float *p, float v) { *p = v; }
__device__ __forceinline__ void ad_store(__nv_bfloat16 *p, float v) { *p = __float2bfloat16(v); }
__device__ __forceinline__ void ad_store(__half *p, float v) { *p = __float2half(v); }

// eight 16-bit weights at a 16-byte boundary
__device__ __forceinline__ void ad_w8(const __nv_bfloat16 *p, float (&v)[8]) {
    const uint4 q = __ldg(reinterpret_cast<const uint4 *>(p));
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void ad_w8(const __half *p, float (&v)[8]) {
    const uint4 q = __ldg(reinterpret_cast<const uint4 *>(p));
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

#define AD_THREADS 256

// One CTA per token: x in shared memory, a warp per row of A, then a thread
// per row of B.
template <typename TX, typename TW, typename TO>
__global__ void __launch_bounds__(AD_THREADS) k_adapter_row(AdapterArgs p) {
    extern __shared__ __align__(16) float xs[];   // [lda]
    __shared__ float low[ADAPTER_MAX_RANK];
    const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int a = p.ids[t];
    const bool have = a >= 0 && a < p.n_adapters;
    int rank = 0;
    if (have) rank = p.ranks ? min(max(p.ranks[a], 0), p.rank) : p.rank;
    if (rank > 0) {
        const TX *x = (const TX *)p.x + (int64_t)t * p.ld_x;
        for (int i = threadIdx.x; i < (int)p.lda; i += AD_THREADS) xs[i] = i < p.n_in ? ad_f32(x[i]) : 0.0f;
        __syncthreads();
        const float scale = p.scale[a];
        for (int r = warp; r < p.rank; r += AD_THREADS / 32) {
            float acc[8] = {};
            if (r < rank) {
                const TW *ar = (const TW *)p.a + ((int64_t)a * p.rank + r) * p.lda;
                for (int i = 8 * lane; i < (int)p.lda; i += 256) {
                    float w[8];
                    ad_w8(ar + i, w);
#pragma unroll
                    for (int c = 0; c < 8; ++c) acc[c] = fmaf(w[c], xs[i + c], acc[c]);
                }
            }
            const float v = warp_sum(((acc[0] + acc[1]) + (acc[2] + acc[3])) + ((acc[4] + acc[5]) + (acc[6] + acc[7])));
            if (lane == 0) low[r] = v * scale;
        }
        __syncthreads();
    }
    const TO *y = (const TO *)p.y + (int64_t)t * p.ld_y;
    TO *out = (TO *)p.out + (int64_t)t * p.ld_out;
    for (int o = threadIdx.x; o < p.n_out; o += AD_THREADS) {
        float acc = 0.0f;
        if (rank > 0) {
            const TW *br = (const TW *)p.b + ((int64_t)a * p.n_out + o) * p.rank;
            for (int r = 0; r < rank; r += 8) {
                float w[8];
                ad_w8(br + r, w);
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (r + c < rank) acc = fmaf(w[c], low[r + c], acc);
            }
        }
        ad_store(out + o, p.y ? ad_f32(y[o]) + acc : acc);
    }
}

template <typename TX, typename TW, typename TO>
static cudaError_t adapters_go(const AdapterArgs &p, cudaStream_t s) {
    const size_t smem = sizeof(float) * (size_t)p.lda;
    if (smem > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(k_adapter_row<TX, TW, TO>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    k_adapter_row<TX, TW, TO><<<p.n_tok, AD_THREADS, smem, s>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_adapters(const AdapterArgs &p, int dt_x, int dt_w, int dt_out, cudaStream_t s) {
    if (p.n_tok == 0 || p.n_out == 0) return cudaSuccess;
    if (dt_x == DT_F32 && dt_out == DT_F32) {
        if (dt_w == DT_BF16) return adapters_go<float, __nv_bfloat16, float>(p, s);
        if (dt_w == DT_F16) return adapters_go<float, __half, float>(p, s);
    }
    if (dt_x == DT_BF16 && dt_w == DT_BF16) {
        if (dt_out == DT_BF16) return adapters_go<__nv_bfloat16, __nv_bfloat16, __nv_bfloat16>(p, s);
        if (dt_out == DT_F32) return adapters_go<__nv_bfloat16, __nv_bfloat16, float>(p, s);
    }
    if (dt_x == DT_F16 && dt_w == DT_F16) {
        if (dt_out == DT_F16) return adapters_go<__half, __half, __half>(p, s);
        if (dt_out == DT_F32) return adapters_go<__half, __half, float>(p, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace moe
